"""Differentiable ops of the package.

CUDA bf16 tensors run the hand-written sm_100a kernels (``csrc/``) through ctypes; anything else (CPU tensors,
fp32) takes a plain PyTorch implementation of the same math, which is also what the numerics tests compare the
kernels against.  There is no eager fallback for CUDA bf16: a missing library raises.

Parameter gradients of these ops are written by the ops themselves (into ``param.main_grad`` when the parameter
has one, an fp32 accumulation buffer, else into ``param.grad``) rather than returned to autograd.  That lets the
weight-gradient GEMM accumulate in fp32 in its epilogue and lets zero-bubble schedules postpone it: while a
:class:`pippy_b200.backward.defer_weight_grads` context is active the weight-gradient work is queued instead of
run.
"""
from __future__ import annotations

import contextlib
import math
from typing import Optional, Tuple, Union

import torch
import torch.nn.functional as F

from ..backward import current_deferral
from . import _lib
from .gemm import ACT_GELU_TANH, ACT_NONE, gemm


def _use_kernels(*tensors: torch.Tensor) -> bool:
    t = tensors[0]
    return t.is_cuda and t.dtype == torch.bfloat16


def _on_device_of(t: torch.Tensor):
    """Launches go to the current device's stream: makes ``t``'s device the current one where it is not."""
    if t.device.index == torch._C._cuda_getDevice():
        return _NOWHERE_ELSE
    return torch.cuda.device(t.device)


_NOWHERE_ELSE = contextlib.nullcontext()


def _no_second_derivative(what: str) -> None:
    """In a backward: gradients are only recorded there when the caller asked for a graph of them."""
    if torch.is_grad_enabled():
        raise RuntimeError(f"{what} has no second derivative on the kernel path")


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """``t`` contiguous and starting on a 16-byte boundary, as kernels with 16-byte accesses need it."""
    t = t.contiguous()
    return t.clone() if t.data_ptr() % 16 else t


_SM_COUNT = {}


def sm_count() -> int:
    dev = torch.cuda.current_device()
    n = _SM_COUNT.get(dev)
    if n is None:
        n = torch.cuda.get_device_properties(dev).multi_processor_count
        _SM_COUNT[dev] = n
    return n


# ------------------------------------------------------------------------------------------------
# parameter-gradient plumbing
# ------------------------------------------------------------------------------------------------
def _accumulate_param_grad(param: torch.Tensor, grad: torch.Tensor) -> None:
    mg = getattr(param, "main_grad", None)
    if mg is not None:
        if grad.dtype == torch.bfloat16 and mg.dtype == torch.float32 and grad.is_cuda and grad.numel() % 8 == 0 and \
                mg.is_contiguous() and mg.data_ptr() % 16 == 0:  # the kernel adds 16 bytes at a time, row by row
            _lib.check(
                _lib.lib().pb_accum_bf16_into_f32(_lib.addr(mg), _lib.addr(_aligned(grad)), grad.numel(),
                                                  _lib.stream_addr()),
                "pb_accum_bf16_into_f32",
            )
        else:
            mg.add_(grad.to(mg.dtype).view_as(mg))
    elif param.grad is None:
        param.grad = grad.to(param.dtype).view_as(param).clone()
    else:
        param.grad.add_(grad.to(param.dtype).view_as(param))


def _run_or_defer(fn) -> None:
    q = current_deferral()
    if q is not None:
        q.defer(fn)
    else:
        fn()


# ------------------------------------------------------------------------------------------------
# linear
# ------------------------------------------------------------------------------------------------
def _wgrad(dy2: torch.Tensor, x2: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor]) -> None:
    mg = getattr(weight, "main_grad", None)
    if mg is not None and mg.dtype == torch.float32:
        gemm(dy2, x2, a_mn=True, b_mn=True, out=mg.view(weight.shape), accumulate=True)
    else:
        dw = gemm(dy2, x2, a_mn=True, b_mn=True)
        _accumulate_param_grad(weight, dw)
    if bias is not None and bias.requires_grad:
        bmg = getattr(bias, "main_grad", None)
        if bmg is not None and bmg.dtype == torch.float32:
            target = bmg
        else:
            target = torch.zeros(bias.shape, dtype=torch.float32, device=bias.device)
        _lib.check(
            _lib.lib().pb_colsum_bf16(_lib.addr(dy2), _lib.addr(target), dy2.shape[0],
                                      dy2.shape[1], dy2.stride(0), _lib.stream_addr()),
            "pb_colsum_bf16",
        )
        if target is not bmg:
            _accumulate_param_grad(bias, target)


class _LinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act: int):
        x2 = x.reshape(-1, x.shape[-1])
        if not x2.is_contiguous():
            x2 = x2.contiguous()
        res2 = None
        if residual is not None:
            res2 = residual.reshape(-1, residual.shape[-1])
            if not res2.is_contiguous():
                res2 = res2.contiguous()
        aux = None
        if act == ACT_GELU_TANH and (x.requires_grad or weight.requires_grad):
            aux = torch.empty(x2.shape[0], weight.shape[0], device=x.device, dtype=torch.bfloat16)
        y = gemm(x2, weight, bias=bias, residual=res2, act=act, aux=aux)
        weight._pb_direct_grad = True
        if bias is not None:
            bias._pb_direct_grad = True
        # Parameters ride on ctx, not in save_for_backward: saved tensors pass through the saved-tensor hooks of
        # activation checkpointing, which hand the backward a detached stand-in without `main_grad` or
        # `requires_grad`, and the weight gradient would be written to an object nobody reads.
        ctx.save_for_backward(x2, aux)
        ctx.weight = weight
        ctx.bias = bias
        ctx.act = act
        ctx.has_residual = residual is not None
        ctx.res_shape = residual.shape if residual is not None else None
        ctx.x_shape = x.shape
        # 2-D in, 2-D out: the result is returned as allocated, never as a view made in here (autograd refuses
        # in-place changes, such as the rotary embedding of a qkv projection, to views created inside a Function)
        return y

    @staticmethod
    def backward(ctx, dy):
        x2, aux = ctx.saved_tensors
        weight, bias = ctx.weight, ctx.bias
        dy2 = dy.reshape(-1, dy.shape[-1])
        if not dy2.is_contiguous():
            dy2 = dy2.contiguous()
        dres = dy.reshape(ctx.res_shape) if ctx.has_residual else None
        if ctx.act == ACT_GELU_TANH:
            dpre = torch.empty_like(dy2)
            _lib.check(
                _lib.lib().pb_gelu_bwd(_lib.addr(dy2), _lib.addr(aux), _lib.addr(dpre), dy2.numel(),
                                       _lib.stream_addr()),
                "pb_gelu_bwd",
            )
            dy2 = dpre
        dx = None
        if ctx.needs_input_grad[0]:
            dx = gemm(dy2, weight, b_mn=True).view(ctx.x_shape)
        if weight.requires_grad:
            _run_or_defer(lambda: _wgrad(dy2, x2, weight, bias))
        return dx, None, None, dres, None


def linear(x, weight, bias=None, residual=None, activation: Optional[str] = None):
    """``act(x @ weight.T + bias) + residual`` with everything after the GEMM fused into its epilogue."""
    if _use_kernels(x):
        act = ACT_GELU_TANH if activation == "gelu_tanh" else ACT_NONE
        if activation not in (None, "gelu_tanh"):
            raise ValueError(f"unsupported fused activation {activation!r}")
        y = _LinearFn.apply(x, weight, bias, residual, act)
        return y if x.dim() == 2 else y.view(*x.shape[:-1], weight.shape[0])
    y = F.linear(x, weight, bias)
    if activation == "gelu_tanh":
        y = F.gelu(y, approximate="tanh")
    elif activation is not None:
        raise ValueError(f"unsupported fused activation {activation!r}")
    if residual is not None:
        y = y + residual
    return y


# ------------------------------------------------------------------------------------------------
# normalisation
# ------------------------------------------------------------------------------------------------
def _norm_scratch(H: int, device) -> torch.Tensor:
    """Partial sums that the norm backward's two kernels hand over: each call's own, since another stream, a captured
    graph or another thread may be between the same two kernels."""
    n = int(_lib.lib().pb_norm_bwd_scratch_floats(H, sm_count()))
    return torch.empty(n, dtype=torch.float32, device=device)


_lib_scratch_restype_set = False


def _ensure_restypes():
    global _lib_scratch_restype_set
    if not _lib_scratch_restype_set:
        _lib.lib().pb_norm_bwd_scratch_floats.restype = _lib.c_ll
        _lib_scratch_restype_set = True


class _NormFn(torch.autograd.Function):
    """``fork=True`` also returns the input itself as a second output: the caller feeds THAT to the residual
    branch, so both gradients of the tensor arrive here and the backward kernel adds the residual one to dx
    (autograd would otherwise sum them with an elementwise kernel of its own)."""

    @staticmethod
    def forward(ctx, x, weight, bias, eps: float, layer: bool, fork: bool):
        _ensure_restypes()
        H = x.shape[-1]
        x2 = x.reshape(-1, H)
        if not x2.is_contiguous():
            x2 = x2.contiguous()
        T = x2.shape[0]
        y = torch.empty_like(x2)
        rstd = torch.empty(T, dtype=torch.float32, device=x.device)
        mean = torch.empty(T, dtype=torch.float32, device=x.device) if layer else None
        _lib.check(
            _lib.lib().pb_norm_fwd(_lib.addr(x2), _lib.addr(weight), _lib.addr(bias), _lib.addr(y), _lib.addr(mean),
                                   _lib.addr(rstd), T, H, eps,
                                   int(layer), _lib.stream_addr()),
            "pb_norm_fwd",
        )
        ctx.save_for_backward(x2, mean, rstd)
        ctx.weight = weight  # not a saved tensor: see _LinearFn.forward
        weight._pb_direct_grad = True
        if bias is not None:
            bias._pb_direct_grad = True
        ctx.bias = bias
        ctx.layer = layer
        ctx.x_shape = x.shape
        ctx.set_materialize_grads(False)  # an unused branch of the fork arrives as None, not as a tensor of zeros
        if fork:
            return y.view(x.shape), x
        return y.view(x.shape)

    @staticmethod
    def backward(ctx, dy, dres=None):
        x2, mean, rstd = ctx.saved_tensors
        weight, bias = ctx.weight, ctx.bias
        T, H = x2.shape
        if dy is None:  # only the residual branch was used
            return dres, None, None, None, None, None
        dy2 = dy.reshape(T, H)
        if not dy2.is_contiguous():
            dy2 = dy2.contiguous()
        if dres is not None:
            dres = dres.reshape(T, H)
            if dres.dtype != x2.dtype:
                dres = dres.to(x2.dtype)
            if not dres.is_contiguous():
                dres = dres.contiguous()
        dx = torch.empty_like(x2)
        wmg = getattr(weight, "main_grad", None)
        use_main = wmg is not None and wmg.dtype == torch.float32
        dw = wmg if use_main else torch.empty(H, dtype=torch.float32, device=x2.device)
        db = None
        if ctx.layer:
            bmg = getattr(bias, "main_grad", None)
            db = bmg if (use_main and bmg is not None) else torch.empty(H, dtype=torch.float32, device=x2.device)
        scratch = _norm_scratch(H, x2.device)
        _lib.check(
            _lib.lib().pb_norm_bwd_res(_lib.addr(dy2), _lib.addr(x2), _lib.addr(weight), _lib.addr(mean),
                                       _lib.addr(rstd), _lib.addr(dres), _lib.addr(dx), _lib.addr(dw), _lib.addr(db),
                                       None, None, int(use_main), _lib.addr(scratch), T, H,
                                       int(ctx.layer), sm_count(), _lib.stream_addr()),
            "pb_norm_bwd_res",
        )
        if not use_main:
            _accumulate_param_grad(weight, dw)
            if ctx.layer:
                _accumulate_param_grad(bias, db)
        return dx.view(ctx.x_shape), None, None, None, None, None


def rms_norm_fork(x, weight, eps: float = 1e-5):
    """``(rms_norm(x), x)`` for the pre-norm residual pattern ``x + f(norm(x))``: use the second result as the
    residual operand.  On the kernel path the gradient that comes back through it is added to the norm's input
    gradient inside the norm-backward kernel."""
    if _use_kernels(x):
        return _NormFn.apply(x, weight, None, eps, False, True)
    return rms_norm(x, weight, eps), x


def rms_norm(x, weight, eps: float = 1e-5):
    if _use_kernels(x):
        return _NormFn.apply(x, weight, None, eps, False, False)
    xf = x.float()
    y = xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps)
    return (y * weight.float()).to(x.dtype)


def layer_norm(x, weight, bias, eps: float = 1e-5):
    if _use_kernels(x):
        return _NormFn.apply(x, weight, bias, eps, True, False)
    return F.layer_norm(x, (x.shape[-1],), weight, bias, eps)


# ------------------------------------------------------------------------------------------------
# activations
# ------------------------------------------------------------------------------------------------
class _SwiGLUFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gu, row_limit=None):
        F2 = gu.shape[-1]
        g2 = gu.reshape(-1, F2)
        if not g2.is_contiguous():
            g2 = g2.contiguous()
        out = torch.empty(g2.shape[0], F2 // 2, device=gu.device, dtype=gu.dtype)
        _lib.check(
            _lib.lib().pb_swiglu_fwd(_lib.addr(g2), _lib.addr(out), g2.shape[0], F2 // 2,
                                     _lib.addr(row_limit), _lib.stream_addr()),
            "pb_swiglu_fwd",
        )
        ctx.save_for_backward(g2)
        ctx.row_limit = row_limit
        ctx.shape = gu.shape
        return out.view(*gu.shape[:-1], F2 // 2)

    @staticmethod
    def backward(ctx, dout):
        (g2,) = ctx.saved_tensors
        d2 = dout.reshape(g2.shape[0], -1)
        if not d2.is_contiguous():
            d2 = d2.contiguous()
        dgu = torch.empty_like(g2)
        _lib.check(
            _lib.lib().pb_swiglu_bwd(_lib.addr(d2), _lib.addr(g2), _lib.addr(dgu), g2.shape[0],
                                     g2.shape[1] // 2, _lib.addr(ctx.row_limit), _lib.stream_addr()),
            "pb_swiglu_bwd",
        )
        return dgu.view(ctx.shape), None


def swiglu(gate_up, row_limit=None):
    """``silu(gate) * up`` for ``gate_up = [..., gate | up]`` (two equal halves on the last dim).  ``row_limit``
    (an int32 device scalar, kernel path only) restricts the work to the first ``row_limit`` rows of a buffer that
    is sized for a capacity; the other rows of the result (and of the gradient) are left as allocated."""
    if _use_kernels(gate_up):
        return _SwiGLUFn.apply(gate_up, row_limit)
    g, u = gate_up.chunk(2, dim=-1)
    return F.silu(g) * u


# ------------------------------------------------------------------------------------------------
# RoPE + attention
# ------------------------------------------------------------------------------------------------
def rope_tables(seq_len: int, head_dim: int, theta: float, device) -> Tuple[torch.Tensor, torch.Tensor]:
    inv = 1.0 / (theta ** (torch.arange(0, head_dim, 2, dtype=torch.float32, device=device) / head_dim))
    ang = torch.outer(torch.arange(seq_len, dtype=torch.float32, device=device), inv)
    return ang.cos().contiguous(), ang.sin().contiguous()


def _rope_inplace(buf: torch.Tensor, cos, sin, T: int, S: int, n_heads: int, D: int, sign: float) -> None:
    _lib.check(
        _lib.lib().pb_rope(_lib.addr(buf), _lib.addr(cos), _lib.addr(sin), T, S,
                           n_heads, D, buf.stride(0), sign,
                           _lib.stream_addr()),
        "pb_rope",
    )


def _rope_ref(x, cos, sin):  # x: [B, S, H, D]
    d2 = x.shape[-1] // 2
    a, b = x[..., :d2].float(), x[..., d2:].float()
    c, s = cos[None, :, None, :], sin[None, :, None, :]
    return torch.cat([a * c - b * s, b * c + a * s], dim=-1).to(x.dtype)


def flash_forward(q, k, v, B, S, Hq, Hkv, D, scale, causal=True):
    """Raw kernel call: q/k/v are 2-D views [B*S, heads*D] (unit inner stride); returns (o [B*S, Hq*D], lse)."""
    o = torch.empty(B * S, Hq * D, device=q.device, dtype=torch.bfloat16)
    lse = torch.empty(B, Hq, S, device=q.device, dtype=torch.float32)
    _lib.check(
        _lib.lib().pb_flash_fwd(_lib.addr(q), _lib.addr(k), _lib.addr(v), _lib.addr(o), _lib.addr(lse), B,
                                S, Hq, Hkv, D,
                                q.stride(0), k.stride(0), v.stride(0),
                                o.stride(0), scale, int(causal),
                                _lib.err_addr(q.device), _lib.stream_addr()),
        "pb_flash_fwd",
    )
    return o, lse


def flash_backward(do, q, k, v, o, lse, B, S, Hq, Hkv, D, scale, causal=True, dqkv: Optional[torch.Tensor] = None):
    """Raw kernel call: returns (dq, dk, dv) as views into one packed [B*S, (Hq + 2 Hkv) * D] buffer."""
    T = B * S
    if dqkv is None:
        dqkv = torch.empty(T, (Hq + 2 * Hkv) * D, device=q.device, dtype=torch.bfloat16)
    dq = dqkv[:, : Hq * D]
    dk = dqkv[:, Hq * D : (Hq + Hkv) * D]
    dv = dqkv[:, (Hq + Hkv) * D :]
    delta = torch.empty(B, Hq, S, device=q.device, dtype=torch.float32)
    _lib.check(
        _lib.lib().pb_flash_bwd(_lib.addr(do), _lib.addr(q), _lib.addr(k), _lib.addr(v), _lib.addr(o), _lib.addr(lse),
                                _lib.addr(delta), _lib.addr(dq), _lib.addr(dk), _lib.addr(dv), B,
                                S, Hq, Hkv, D,
                                q.stride(0), k.stride(0), v.stride(0),
                                o.stride(0), do.stride(0), dqkv.stride(0),
                                scale, int(causal), _lib.err_addr(q.device),
                                _lib.stream_addr()),
        "pb_flash_bwd",
    )
    return dq, dk, dv, dqkv


class _RopeAttentionFn(torch.autograd.Function):
    """qkv [B*S, (Hq + 2 Hkv) * D] -> attention output [B*S, Hq * D].

    RoPE is applied to the q and k columns of ``qkv`` IN PLACE (the rotated projection is what the backward needs,
    and a second copy of the largest activation of the layer would be kept for nothing).  The kernel writes through
    a raw pointer, so the tensor's version counter is bumped by hand: a producer that had saved ``qkv`` for its own
    backward gets autograd's usual "modified by an inplace operation" error instead of silently wrong gradients.
    The gradient returned for ``qkv`` is with respect to its value BEFORE the rotation."""

    @staticmethod
    def forward(ctx, qkv, cos, sin, B, S, Hq, Hkv, D, scale, causal):
        T = B * S
        if cos is not None:
            _rope_inplace(qkv, cos, sin, T, S, Hq + Hkv, D, 1.0)
            torch.autograd.graph.increment_version(qkv)
        q = qkv[:, : Hq * D]
        k = qkv[:, Hq * D : (Hq + Hkv) * D]
        v = qkv[:, (Hq + Hkv) * D :]
        o, lse = flash_forward(q, k, v, B, S, Hq, Hkv, D, scale, causal)
        ctx.save_for_backward(qkv, o, lse, cos, sin)
        ctx.cfg = (B, S, Hq, Hkv, D, scale, causal)
        return o

    @staticmethod
    def backward(ctx, do):
        qkv, o, lse, cos, sin = ctx.saved_tensors
        B, S, Hq, Hkv, D, scale, causal = ctx.cfg
        q = qkv[:, : Hq * D]
        k = qkv[:, Hq * D : (Hq + Hkv) * D]
        v = qkv[:, (Hq + Hkv) * D :]
        if not do.is_contiguous():
            do = do.contiguous()
        _, _, _, dqkv = flash_backward(do, q, k, v, o, lse, B, S, Hq, Hkv, D, scale, causal)
        if cos is not None:
            _rope_inplace(dqkv, cos, sin, B * S, S, Hq + Hkv, D, -1.0)
        return dqkv, None, None, None, None, None, None, None, None, None


def rope_attention(qkv, cos, sin, B: int, S: int, Hq: int, Hkv: int, D: int, scale: Optional[float] = None,
                   causal: bool = True):
    """Causal self-attention over a packed projection ``qkv`` of shape ``[B*S, (Hq + 2*Hkv) * D]``
    (q heads, then k heads, then v heads), with rotary embedding of q and k when ``cos``/``sin`` are given.

    On the kernel path (CUDA bf16) the rotation overwrites the q and k columns of ``qkv``: the caller's tensor holds
    the rotated projection afterwards (its version counter is bumped).  Pass a clone to keep the original.  The
    CPU path leaves ``qkv`` untouched."""
    scale = (1.0 / math.sqrt(D)) if scale is None else scale
    if _use_kernels(qkv):
        return _RopeAttentionFn.apply(qkv, cos, sin, B, S, Hq, Hkv, D, scale, causal)
    q = qkv[:, : Hq * D].view(B, S, Hq, D)
    k = qkv[:, Hq * D : (Hq + Hkv) * D].view(B, S, Hkv, D)
    v = qkv[:, (Hq + Hkv) * D :].view(B, S, Hkv, D)
    if cos is not None:
        q, k = _rope_ref(q, cos, sin), _rope_ref(k, cos, sin)
    rep = Hq // Hkv
    k = k.repeat_interleave(rep, dim=2)
    v = v.repeat_interleave(rep, dim=2)
    att = torch.einsum("bqhd,bkhd->bhqk", q.float(), k.float()) * scale
    if causal:
        mask = torch.ones(S, S, dtype=torch.bool, device=qkv.device).tril()
        att = att.masked_fill(~mask, float("-inf"))
    att = att.softmax(-1)
    out = torch.einsum("bhqk,bkhd->bqhd", att, v.float()).to(qkv.dtype)
    return out.reshape(B * S, Hq * D)


# ------------------------------------------------------------------------------------------------
# cross entropy
# ------------------------------------------------------------------------------------------------
class _CrossEntropyFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, vocab: int, reduction: str, ignore_index: int, inplace: bool):
        T, ld = logits.shape
        tgt = targets.reshape(-1).contiguous()
        dev = logits.device
        loss_rows = torch.empty(T, dtype=torch.float32, device=dev)
        # the gradient is formed with the loss, where anyone wants it (`inplace` promises it in `logits`)
        dlogits = logits if inplace else (torch.empty_like(logits) if ctx.needs_input_grad[0] else None)
        n_valid = torch.empty((), dtype=torch.float32, device=dev) if reduction == "mean" else None
        loss = torch.empty((), dtype=torch.float32, device=dev)
        _lib.check(
            _lib.lib().pb_xent(_lib.addr(logits), _lib.addr(dlogits), _lib.addr(tgt), _lib.addr(loss_rows),
                               _lib.addr(n_valid), _lib.addr(loss), T, vocab,
                               logits.stride(0), ignore_index, _lib.stream_addr()),
            "pb_xent",
        )
        ctx.save_for_backward(dlogits)
        return loss

    @staticmethod
    def backward(ctx, dloss):
        (dlogits,) = ctx.saved_tensors
        scale = dloss.to(torch.float32).reshape(1).contiguous()
        _lib.check(
            _lib.lib().pb_scale_bf16(_lib.addr(dlogits), _lib.addr(scale), dlogits.numel(),
                                     _lib.stream_addr()),
            "pb_scale_bf16",
        )
        return dlogits, None, None, None, None, None


def cross_entropy(logits, targets, vocab_size: Optional[int] = None, reduction: str = "mean",
                  ignore_index: int = -100, inplace: bool = False):
    """Softmax cross-entropy over ``logits [T, V_padded]``; columns at or beyond ``vocab_size`` are padding.
    With ``inplace=True`` the gradient overwrites ``logits`` (saves one [T, V] buffer)."""
    if reduction not in ("mean", "sum"):
        raise ValueError("reduction must be 'mean' or 'sum'")
    logits2 = logits.reshape(-1, logits.shape[-1])
    V = logits2.shape[-1] if vocab_size is None else vocab_size
    if _use_kernels(logits2):
        if not logits2.is_contiguous():
            logits2 = logits2.contiguous()
        return _CrossEntropyFn.apply(logits2, targets, V, reduction, ignore_index, inplace)
    return F.cross_entropy(logits2[:, :V].float(), targets.reshape(-1), reduction=reduction, ignore_index=ignore_index)


# ------------------------------------------------------------------------------------------------
# embedding
# ------------------------------------------------------------------------------------------------
def _embed_wgrad(ids, dout, wte, wpe, S):
    T, H = dout.shape
    wmg = getattr(wte, "main_grad", None)
    dw = wmg if (wmg is not None and wmg.dtype == torch.float32) else torch.zeros(wte.shape, dtype=torch.float32, device=wte.device)
    dp = None
    if wpe is not None:
        pmg = getattr(wpe, "main_grad", None)
        dp = pmg if (pmg is not None and pmg.dtype == torch.float32) else torch.zeros(wpe.shape, dtype=torch.float32, device=wpe.device)
    _lib.check(
        _lib.lib().pb_embed_bwd(_lib.addr(ids), _lib.addr(dout), _lib.addr(dw), _lib.addr(dp), T,
                                H, S, wte.shape[0], _lib.stream_addr()),
        "pb_embed_bwd",
    )
    if dw is not wmg:
        _accumulate_param_grad(wte, dw)
    if wpe is not None and dp is not getattr(wpe, "main_grad", None):
        _accumulate_param_grad(wpe, dp)


class _EmbeddingFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, wte, wpe, S: int):
        flat = ids.reshape(-1).contiguous()
        T, H = flat.numel(), wte.shape[1]
        out = torch.empty(T, H, device=wte.device, dtype=wte.dtype)
        _lib.check(
            _lib.lib().pb_embed_fwd(_lib.addr(flat), _lib.addr(wte), _lib.addr(wpe), _lib.addr(out), T,
                                    H, S, wte.shape[0], _lib.stream_addr()),
            "pb_embed_fwd",
        )
        ctx.save_for_backward(flat)
        wte._pb_direct_grad = True
        if wpe is not None:
            wpe._pb_direct_grad = True
        ctx.params = (wte, wpe)
        ctx.S = S
        return out

    @staticmethod
    def backward(ctx, dout):
        (flat,) = ctx.saved_tensors
        wte, wpe = ctx.params
        d2 = dout.contiguous()
        S = ctx.S
        _run_or_defer(lambda: _embed_wgrad(flat, d2, wte, wpe, S))
        return None, None, None, None


# In the place of a table that a captured graph leaves out, see below.  A leaf on the CPU has no stream.
_NO_STREAM = torch.empty(0, device="cpu", requires_grad=True)
_MADE_ON = "pippy_b200 stream"  # in the metadata of accumulation nodes that captured embeddings made


def _held_elsewhere(table: torch.Tensor, stream: int) -> bool:
    """Whether a graph that was not made on ``stream`` holds the leaf's accumulation node."""
    node = torch.autograd.graph.get_gradient_edge(table).node  # made here where there is none
    if _MADE_ON in node.metadata:
        return node.metadata[_MADE_ON] != stream
    node.metadata[_MADE_ON] = stream
    del node  # a node that nobody else holds ends here, and what was noted on it
    node = torch.autograd.graph.get_gradient_edge(table).node
    return node.metadata.pop(_MADE_ON, None) is not None


def _captured_inputs(tables):
    """Under capture, the leaves that the op below is a function of in autograd.  They are the tables that it writes
    gradients for, whose accumulation nodes ``backward(inputs=...)``, hooks and wrappers that count ready parameters go by.

    Such a node belongs to the stream on which the first of the graphs that hold it was made, and a backward waits for
    the streams of the nodes that it reaches.  Captured, it cannot wait for a stream outside its capture: that ends the
    process.  So a captured graph leaves a table out whose node a graph of another stream holds."""
    stream = torch.cuda.current_stream().cuda_stream
    kept = [t for t in tables if not _held_elsewhere(t, stream)]
    return kept if len(kept) == len(tables) else kept + [_NO_STREAM]


def _note_stream(leaves) -> None:
    """After the graph of ``leaves`` is made: a node of this capture serves the capture's later embeddings too."""
    for t in leaves:
        if t is not _NO_STREAM:
            torch.autograd.graph.get_gradient_edge(t).node.metadata[_MADE_ON] = torch.cuda.current_stream().cuda_stream


class _SortedEmbeddingFn(torch.autograd.Function):
    """On the device of the tables.  ``leaves``: those that are trained, under capture see :func:`_captured_inputs`; their
    gradients are written by the kernels."""

    @staticmethod
    def forward(ctx, ids, tables, positions, S: int, scale: float, *leaves):
        wte, wpe = tables
        T, H = ids.numel(), wte.shape[1]
        table, ptable = wte, wpe
        if wte.data_ptr() % 16 or not wte.is_contiguous():
            table = _aligned(wte.detach())
        if wpe is not None and (wpe.data_ptr() % 16 or not wpe.is_contiguous()):
            ptable = _aligned(wpe.detach())
        out = torch.empty(T, H, device=wte.device, dtype=wte.dtype)
        _lib.check(
            _lib.lib().pb_embed_scaled_fwd(ids.data_ptr(), table.data_ptr(), _lib.addr(ptable), _lib.addr(positions),
                                           out.data_ptr(), T, H, S, wte.shape[0], 0 if wpe is None else wpe.shape[0], scale,
                                           _lib.err_addr(wte.device), _lib.stream_addr()),
            "pb_embed_scaled_fwd",
        )
        ctx.save_for_backward(ids, positions)
        wte._pb_direct_grad = True
        if wpe is not None:
            wpe._pb_direct_grad = True
        ctx.cfg = (wte, wpe, S, scale)  # parameters are not saved tensors: see _LinearFn.forward
        return out

    @staticmethod
    def backward(ctx, dout):
        _no_second_derivative("embedding with sorted gradients")
        ids, positions = ctx.saved_tensors
        dout = _aligned(dout)
        if current_deferral() is None:
            _embed_sorted_wgrad(ids, positions, dout, *ctx.cfg)
        else:
            cfg = ctx.cfg
            _run_or_defer(lambda: _embed_sorted_wgrad(ids, positions, dout, *cfg))
        return (None,) * len(ctx.needs_input_grad)


def _sorted_grad_target(p):
    """Where the kernel puts a table's gradient, and whether it writes it whole, in the table's type, or adds it in fp32."""
    if p is None or not p.requires_grad:
        return None, False
    mg = getattr(p, "main_grad", None)
    if mg is None or mg.dtype != torch.float32:
        return torch.empty(p.shape, dtype=p.dtype, device=p.device), True
    if mg.is_contiguous() and mg.data_ptr() % 16 == 0:
        return mg, False
    return torch.zeros(p.shape, dtype=torch.float32, device=p.device), False


def _embed_sorted_wgrad(ids, positions, dout, wte, wpe, S, scale):
    T, H = dout.shape
    lib = _lib.lib()
    with _on_device_of(dout):
        (gw, write_w), (gp, write_p) = targets = _sorted_grad_target(wte), _sorted_grad_target(wpe)
        # one launch for both tables, unless one has an fp32 buffer and the other one has none
        together = gw is None or gp is None or write_w == write_p
        for a, b, write in ((gw, gp, write_w or write_p),) if together else ((gw, None, write_w), (None, gp, write_p)):
            scratch = torch.empty(lib.pb_embed_sorted_scratch(T, H, (a is not None) + (b is not None)), dtype=torch.uint8,
                                  device=dout.device)
            _lib.check(
                lib.pb_embed_sorted_bwd(ids.data_ptr(), _lib.addr(positions), dout.data_ptr(), _lib.addr(a), _lib.addr(b), T, H, S,
                                        wte.shape[0], 0 if wpe is None else wpe.shape[0], scale, int(write),
                                        scratch.data_ptr(), _lib.stream_addr()),
                "pb_embed_sorted_bwd",
            )
        for p, (g, _) in zip((wte, wpe), targets):
            mg = getattr(p, "main_grad", None)
            if g is None or g is mg:
                continue
            if mg is None and p.grad is None:
                p.grad = g
            else:
                _accumulate_param_grad(p, g)


def embedding(ids, wte, wpe=None, seq_len: Optional[int] = None, scale: float = 1.0,
              positions: Optional[torch.Tensor] = None, sorted_grad: bool = False):
    """``scale * wte[ids] (+ wpe[position])`` flattened to ``[B*S, H]``; position of token t is ``t % seq_len``, or
    ``positions[t]`` where given (a :class:`PackedLayout`'s, -1 adds nothing).

    The tables' gradients are fp32 scatter-adds, whose order changes from run to run, unless ``sorted_grad`` is set:
    then, and always with a ``scale`` or ``positions``, tokens are sorted first and the rows of a token added in their
    order, the same bits on every run.  On that path ids outside ``wte`` and positions beyond ``wpe`` give zeros and
    set the device error word (:func:`pippy_b200.ops._lib.check_device_errors`).  Captured while a graph made on another
    stream (an eager one) holds a table's accumulation node, the graph leaves that table out: its gradient is written, but
    ``backward(inputs=...)`` does not count it and hooks on it do not run."""
    S = ids.shape[-1] if seq_len is None else seq_len
    plain = scale == 1.0 and positions is None
    if positions is not None:
        if wpe is None:
            raise ValueError("positions were given without a table of positions")
        if positions.numel() != ids.numel() or positions.device != ids.device or positions.is_floating_point():
            raise ValueError(f"positions: one integer for each of {ids.numel()} ids, on their device; got "
                             f"{tuple(positions.shape)} {positions.dtype} on {positions.device}")
    if wte.is_cuda and wte.dtype == torch.bfloat16:
        if plain and not sorted_grad:
            # autograd only tracks the op if some input requires grad; tie it to the table
            return _EmbeddingFn.apply(ids, wte, wpe, S)
        if ids.device != wte.device or ids.is_floating_point():
            raise ValueError(f"ids: integers on {wte.device}, got {ids.dtype} on {ids.device}")
        if wte.dim() != 2 or wte.shape[1] % 8 or (wpe is not None and (
                wpe.shape[1:] != wte.shape[1:] or wpe.dtype != wte.dtype or wpe.device != wte.device)):
            raise ValueError("tables: [rows, H] of one type on one device, H a multiple of 8")
        if wpe is wte:
            raise ValueError("one tensor as both tables: their gradients are written at the same time")
        trained = [w for w in (wte, wpe) if w is not None and w.requires_grad]
        if not all(w.is_leaf for w in trained):
            raise ValueError("tables that require gradients have to be leaves: the kernels write their gradients")
        if positions is not None:
            if positions.dtype != torch.int32 or not positions.is_contiguous():
                # positions beyond 32 bits would wrap to ones that seem to fit
                positions = positions.long().clamp(-1, 2 ** 31 - 1).to(torch.int32).contiguous()
        if ids.dtype != torch.int64 or not ids.is_contiguous():
            ids = ids.long().contiguous()
        S = S if ids.numel() else 1
        with _on_device_of(wte):
            captured = torch.cuda.is_current_stream_capturing() and torch.is_grad_enabled()
            leaves = _captured_inputs(trained) if captured else trained
            out = _SortedEmbeddingFn.apply(ids, (wte, wpe), positions, S, float(scale), *leaves)
            if captured:
                _note_stream(leaves)
        return out
    if plain:
        out = F.embedding(ids.reshape(-1), wte)
        if wpe is not None:
            pos = torch.arange(ids.numel(), device=ids.device) % S
            out = out + F.embedding(pos, wpe)
        return out
    wide = torch.promote_types(wte.dtype, torch.float32)
    out = F.embedding(ids.reshape(-1), wte).to(wide) * scale
    if wpe is not None:
        pos = (torch.arange(ids.numel(), device=ids.device) % S) if positions is None else positions.reshape(-1).long()
        out = out + torch.where((pos >= 0).unsqueeze(1), F.embedding(pos.clamp(min=0), wpe).to(wide), 0.0)
    return out.to(wte.dtype)


# ------------------------------------------------------------------------------------------------
# packed documents
# ------------------------------------------------------------------------------------------------
class PackedLayout:
    """Where the documents of a packed batch lie (:func:`packed_layout`).  One layout serves every layer of a batch, forward
    and backward.

    ``positions``: int32 ``[rows * tokens_per_row]``, each token's place in its document, -1 in padding."""

    def __init__(self, lengths: torch.Tensor, tokens_per_row: int, positions: torch.Tensor, tables=None, most=(0, 0)):
        self.lengths, self.tokens_per_row, self.positions = lengths, tokens_per_row, positions
        self.rows = lengths.shape[0]
        self.total = self.rows * tokens_per_row
        self.device = lengths.device
        # kernel path: the tiles of 128 and of 256 rows (4 ints each, room for `most` of them), then for both tables 4 ints:
        # how many there are, how many before the half-filled ones, how many before the padding
        self._tables, self._most = tables, most

    def tiles(self, rows: int) -> Tuple[torch.Tensor, torch.Tensor]:
        """``(tiles, counts)`` of ``rows`` = 128 or 256 rows, for inspection: ``[n, 4]`` of document start, document
        length, number of the tile in it, 1 for padding."""
        first, n = (0, self._most[0]) if rows == 128 else (self._most[0], self._most[1])
        counts = self._tables[4 * sum(self._most) :].view(2, 4)[0 if rows == 128 else 1]
        return self._tables[4 * first : 4 * (first + n)].view(n, 4), counts

    def _addresses(self):
        """Addresses of the tiles of 128 and of 256 rows and of their counts."""
        base, (n128, n256) = self._tables.data_ptr(), self._most
        return base, base + 16 * n128, base + 16 * (n128 + n256), base + 16 * (n128 + n256) + 16


def packed_layout(lengths: torch.Tensor, tokens_per_row: int) -> PackedLayout:
    """The layout of rows of ``tokens_per_row`` tokens that hold documents one after the other: ``lengths`` is an integer
    tensor ``[rows, documents]`` (or ``[documents]`` for one row); a length may be 0 (rows with fewer documents), and what a
    row has left behind its last document is padding.

    On the GPU this is one kernel: the lengths stay on the device and nothing waits for them.  Lengths that are negative or
    exceed their row are cut to what fits and set the device error word
    (:func:`pippy_b200.ops._lib.check_device_errors`); on the CPU they raise."""
    if lengths.dim() == 1:
        lengths = lengths.unsqueeze(0)
    if lengths.dim() != 2 or lengths.shape[0] < 1 or lengths.is_floating_point() or lengths.is_complex() or \
            lengths.dtype == torch.bool:
        raise ValueError(f"lengths: integers [rows, documents], got {tuple(lengths.shape)} {lengths.dtype}")
    rows, docs = lengths.shape
    S = int(tokens_per_row)
    if S < 1 or rows * S >= 2 ** 30 or rows * (docs + 1) >= 2 ** 30:
        raise ValueError(f"{rows} rows of {S} tokens with {docs} documents each: between 1 and 2^30 - 1 of both")
    if not lengths.is_cuda:
        if docs and (bool((lengths < 0).any()) or int(lengths.long().sum(1).max()) > S):
            raise ValueError(f"document lengths are negative or exceed the row of {S} tokens")
        ends = lengths.long().cumsum(1)
        t = torch.arange(S).expand(rows, S).contiguous()
        positions = torch.full((rows, S), -1, dtype=torch.int32)
        if docs:
            doc = torch.searchsorted(ends, t, right=True)
            starts = torch.cat([torch.zeros_like(ends[:, :1]), ends], 1)
            positions = torch.where(t < ends[:, -1:], t - starts.gather(1, doc), -1).int()
        return PackedLayout(lengths, S, positions.reshape(-1))
    with _on_device_of(lengths):
        # lengths beyond 32 bits would wrap to ones that seem to fit
        given = (lengths if lengths.dtype == torch.int32 else lengths.long().clamp(-1, 2 ** 31 - 1).to(torch.int32)).contiguous()
        segments = rows * (docs + 1)
        spare = min(segments, rows * S)
        n128, n256 = rows * S // 128 + spare, rows * S // 256 + spare
        # one buffer: tiles of 4 ints, counts, segments of 2 ints (an even number of them), positions
        first = 4 * (n128 + n256) + 8 + (2 * segments + 3) // 4 * 4
        buf = torch.empty(first + rows * S, dtype=torch.int32, device=lengths.device)
        layout = PackedLayout(given, S, buf[first:], buf[: 4 * (n128 + n256) + 8], (n128, n256))
        t128, t256, counts, _ = layout._addresses()
        _lib.check(
            _lib.lib().pb_packed_layout(given.data_ptr(), rows, docs, S, t128 + 4 * first, counts + 32, t128, n128, t256,
                                        n256, counts, _lib.err_addr(lengths.device), _lib.stream_addr()),
            "pb_packed_layout",
        )
    return layout


class _PackedAttentionFn(torch.autograd.Function):
    """As :class:`_RopeAttentionFn`, over documents.  Without ``inplace`` the rotated q and k are a tensor of their own and
    ``qkv`` stays as it is; its v columns are read in place either way."""

    @staticmethod
    def forward(ctx, qkv, cos, sin, layout, Hq, Hkv, D, scale, causal, inplace):
        # q, k and v are columns of qkv (of qk): addresses instead of views, which cost more than the launch in small calls
        T, nq, nk = layout.total, Hq * D, Hkv * D
        lib, err = _lib.lib(), _lib.err_addr(qkv.device)
        with _on_device_of(qkv):
            stream = _lib.stream_addr()
            lse = torch.empty(Hq * T + 1, device=qkv.device, dtype=torch.float32)  # and the forward's counter
            counter = lse.data_ptr() + 4 * Hq * T
            qk = qkv
            if cos is not None:
                if not inplace:
                    qk = torch.empty(T, nq + nk, device=qkv.device, dtype=qkv.dtype)
                _lib.check(
                    lib.pb_packed_rope(qkv.data_ptr(), qkv.stride(0), qk.data_ptr(), qk.stride(0), cos.data_ptr(),
                                       sin.data_ptr(), layout.positions.data_ptr(), T, Hq + Hkv, D, cos.shape[0],
                                       counter, err, stream),
                    "pb_packed_rope",
                )
                if inplace:
                    torch.autograd.graph.increment_version(qkv)
            o = torch.empty(T, nq, device=qkv.device, dtype=qkv.dtype)
            _, t256, _, counts = layout._addresses()
            q, v, pitch = qk.data_ptr(), qkv.data_ptr() + 2 * (nq + nk), qk.stride(0)
            _lib.check(
                lib.pb_packed_attention_fwd(q, q + 2 * nq, v, o.data_ptr(), lse.data_ptr(), counter,
                                            int(cos is not None), t256, counts, layout._most[1], T, Hq, Hkv, D, pitch,
                                            pitch, qkv.stride(0), nq, scale, int(causal), err, stream),
                "pb_packed_attention_fwd",
            )
        ctx.save_for_backward(qkv, qk, o, lse, cos, sin)
        ctx.cfg = (layout, Hq, Hkv, D, scale, causal)
        return o

    @staticmethod
    def backward(ctx, do):
        _no_second_derivative("packed_attention")
        qkv, qk, o, lse, cos, sin = ctx.saved_tensors
        layout, Hq, Hkv, D, scale, causal = ctx.cfg
        T, nq, nk = layout.total, Hq * D, Hkv * D
        with _on_device_of(qkv):
            do = _aligned(do)
            dqkv = torch.empty(T, nq + 2 * nk, device=qkv.device, dtype=qkv.dtype)
            lib = _lib.lib()
            scratch = torch.empty(lib.pb_packed_attention_bwd_scratch(T, Hq, Hkv, D, layout._most[0]), dtype=torch.uint8,
                                  device=qkv.device)
            t128, _, counts, _ = layout._addresses()
            q, v, d, pitch = qk.data_ptr(), qkv.data_ptr() + 2 * (nq + nk), dqkv.data_ptr(), qk.stride(0)
            _lib.check(
                lib.pb_packed_attention_bwd(
                    do.data_ptr(), q, q + 2 * nq, v, o.data_ptr(), lse.data_ptr(), scratch.data_ptr(), d, d + 2 * nq,
                    d + 2 * (nq + nk), _lib.addr(cos), _lib.addr(sin), 0 if cos is None else cos.shape[0], t128, counts,
                    layout._most[0], layout.positions.data_ptr(), T, Hq, Hkv, D, pitch, pitch, qkv.stride(0), nq, nq,
                    nq + 2 * nk, scale, int(causal), _lib.err_addr(qkv.device),
                    _lib.stream_addr()),
                "pb_packed_attention_bwd",
            )
        return dqkv, None, None, None, None, None, None, None, None, None


def packed_attention(qkv, cos, sin, layout: PackedLayout, Hq: int, Hkv: int, D: int, scale: Optional[float] = None,
                     causal: bool = True, inplace: bool = False):
    """Self-attention inside each document of a packed batch: ``qkv`` is ``[layout.total, (Hq + 2*Hkv) * D]`` (q heads, then k
    heads, then v heads), the result ``[layout.total, Hq * D]``.  Tokens see the tokens of their own document, with
    ``causal`` those up to themselves; padding rows give zeros, in the result and in the gradient, whatever they hold.
    Heads of q share the k and v heads in groups of ``Hq // Hkv``.

    ``cos`` / ``sin`` (fp32 ``[positions, D / 2]``, see :func:`rope_tables`) rotate q and k by the position inside the
    document; their rows have to reach the longest document (on the kernel path longer ones set the device error word and
    stay unrotated from there on, on the CPU they raise).  With ``inplace`` the rotation overwrites the q and k columns
    of ``qkv`` (its version counter is bumped), which saves a tensor of their size; without rotation it means nothing.

    Kernel path (CUDA bf16): D is 64 or 128; sums have a fixed order, the same bits on every run."""
    scale = (1.0 / math.sqrt(D)) if scale is None else float(scale)
    if Hq < 1 or Hkv < 1 or Hq % Hkv:
        raise ValueError(f"{Hq} query heads cannot share {Hkv} key heads evenly")
    if qkv.dim() != 2 or qkv.shape[0] != layout.total or qkv.shape[1] != (Hq + 2 * Hkv) * D:
        raise ValueError(f"qkv: [{layout.total}, {(Hq + 2 * Hkv) * D}] for this layout and these heads, got "
                         f"{tuple(qkv.shape)}")
    if not (scale > 0 and math.isfinite(scale)):
        raise ValueError(f"scale has to be positive and finite, got {scale}")
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin come together")
    for t in () if cos is None else (cos, sin):
        if t.dim() != 2 or t.shape != cos.shape or t.shape[1] != D // 2 or t.dtype != torch.float32 or \
                t.device != qkv.device:
            raise ValueError(f"cos / sin: fp32 [positions, {D // 2}] on {qkv.device}, got {tuple(t.shape)} {t.dtype} on "
                             f"{t.device}")
    if layout.device != qkv.device:
        raise ValueError(f"the layout is on {layout.device}, qkv on {qkv.device}")
    if _use_kernels(qkv):
        if D not in (64, 128):
            raise ValueError(f"the kernels have head sizes 64 and 128, got {D}")
        if qkv.stride(1) != 1 or qkv.stride(0) % 8 or qkv.stride(0) < qkv.shape[1] or qkv.data_ptr() % 16:
            if inplace and cos is not None:
                raise ValueError("inplace needs rows of unit stride that start on 16-byte boundaries")
            qkv = qkv.clone(memory_format=torch.contiguous_format)
        if cos is not None:
            cos, sin = _aligned(cos), _aligned(sin)
        return _PackedAttentionFn.apply(qkv, cos, sin, layout, Hq, Hkv, D, scale, causal, inplace)
    rows, S = layout.rows, layout.tokens_per_row
    pos = layout.positions.view(rows, S).long()
    wide = torch.promote_types(qkv.dtype, torch.float32)
    q, k, v = (t.reshape(rows, S, -1, D).transpose(1, 2).to(wide) for t in qkv.split([Hq * D, Hkv * D, Hkv * D], dim=1))
    if cos is not None:
        if int(pos.max()) >= cos.shape[0]:
            raise ValueError(f"a document of {int(pos.max()) + 1} tokens, cos / sin for {cos.shape[0]}")
        c, s = (t[pos.clamp(min=0)].unsqueeze(1).to(wide) for t in (cos, sin))
        q, k = (torch.cat([a * c - b * s, b * c + a * s], dim=-1) for a, b in (q.chunk(2, -1), k.chunk(2, -1)))
        q, k = q.to(qkv.dtype).to(wide), k.to(qkv.dtype).to(wide)
    k, v = k.repeat_interleave(Hq // Hkv, 1), v.repeat_interleave(Hq // Hkv, 1)
    doc = torch.cumsum(pos == 0, 1)  # a document's tokens follow its first one
    seen = (doc.unsqueeze(2) == doc.unsqueeze(1)) & (pos >= 0).unsqueeze(2) & (pos >= 0).unsqueeze(1)
    if causal:
        seen = seen & (pos.unsqueeze(2) >= pos.unsqueeze(1))
    inside = (pos >= 0).view(rows, 1, S, 1)
    # what padding holds (an Inf, say) must not reach a product
    q, k, v = (torch.where(inside, t, 0.0) for t in (q, k, v))
    att = (q @ k.transpose(2, 3) * scale).masked_fill(~seen.unsqueeze(1), torch.finfo(wide).min).softmax(-1)
    out = torch.where(inside, att @ v, 0.0)
    return out.transpose(1, 2).reshape(rows * S, Hq * D).to(qkv.dtype)


# ------------------------------------------------------------------------------------------------
# dropout
# ------------------------------------------------------------------------------------------------
def _philox_blocks(seed: int, stream: int, block: torch.Tensor) -> torch.Tensor:
    """The eight 16-bit numbers of each numbered block of elements, in 64-bit integer arithmetic."""
    low = 0xFFFFFFFF
    x = [block & low, block >> 32, torch.full_like(block, stream & low), torch.full_like(block, (stream >> 32) & low)]
    k0, k1 = seed & low, (seed >> 32) & low
    for _ in range(10):
        a, b = x[0] * 0xD2511F53, x[2] * 0xCD9E8D57  # modulo 2^64: the shift leaves the upper half's bits in place
        x = [((b >> 32) & low) ^ x[1] ^ k0, b & low, ((a >> 32) & low) ^ x[3] ^ k1, a & low]
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    words = torch.stack(x, 1)
    return torch.stack([words & 0xFFFF, words >> 16], 2).reshape(-1, 8)


def _philox_numbers(seed: int, stream: int, count: int, device) -> torch.Tensor:
    """``count`` 16-bit numbers as ``csrc/dropout.cu`` draws them."""
    return _philox_blocks(seed, stream, torch.arange((count + 7) // 8, device=device)).reshape(-1)[:count]


class _DropoutFn(torch.autograd.Function):
    """The mask is a function of the seed: the backward computes it again.  A seed tensor is a saved tensor, so changing it
    in place between the two is autograd's usual error."""

    @staticmethod
    def forward(ctx, x, residual, seed, seed_value: int, stream: int, threshold: int):
        ctx.save_for_backward(seed)
        ctx.cfg = (seed_value, stream, threshold)
        return _launch_dropout(x, residual, seed, seed_value, stream, threshold)

    @staticmethod
    def backward(ctx, dy):
        (seed,) = ctx.saved_tensors
        dx = None
        if ctx.needs_input_grad[0]:
            if torch.is_grad_enabled():  # linear in dy: its derivative is the same mask once more
                dx = _DropoutFn.apply(dy, None, seed, *ctx.cfg)
            else:
                dx = _launch_dropout(dy, None, seed, *ctx.cfg)
        return dx, dy if ctx.needs_input_grad[1] else None, None, None, None, None


def _launch_dropout(x, residual, seed, seed_value, stream, threshold):
    x = x.contiguous()
    if residual is not None:
        residual = residual.contiguous()
    y = torch.empty_like(x)
    with _on_device_of(x):
        _lib.check(
            _lib.lib().pb_dropout(x.data_ptr(), _lib.addr(residual), y.data_ptr(), x.numel(), _lib.addr(seed),
                                  seed_value, stream, threshold, _lib.stream_addr()),
            "pb_dropout",
        )
    return y


def dropout(x, p: float, seed: Union[int, torch.Tensor], residual: Optional[torch.Tensor] = None, stream: int = 0):
    """``x * mask / (1 - p) (+ residual)``, each element dropped with probability ``p`` (rounded to a multiple of 2^-16; the
    factor uses the rounded value).  The mask is a function of ``(seed, stream, element index)`` by Philox4x32-10 (Salmon et
    al., SC 2011), the same on every device, and is never stored: the backward computes it again.

    ``seed``: an int, or an int64 tensor of one element on ``x``'s device, read when the kernel runs (a captured graph
    draws another mask for another seed in it).  ``stream``: a number from 0 to 2^63 - 1 that keeps the layers of one seed
    apart.  Dropped elements are 0 (or ``residual``) whatever ``x`` holds."""
    threshold = int(math.floor(p * 65536 + 0.5)) if 0.0 <= p <= 1.0 else -1
    if not 0 <= threshold <= 65535:
        raise ValueError(f"p has to be at least 0 and below 1 - 2^-17, got {p}")
    if not 0 <= stream < 2 ** 63:
        raise ValueError(f"stream: 0 to 2^63 - 1, got {stream}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype or residual.device != x.device):
        raise ValueError(f"residual: {tuple(x.shape)} {x.dtype} on {x.device}, got {tuple(residual.shape)} "
                         f"{residual.dtype} on {residual.device}")
    if isinstance(seed, torch.Tensor):
        if seed.dtype != torch.int64 or seed.numel() != 1 or seed.device != x.device:
            raise ValueError(f"seed: one int64 on {x.device}, got {tuple(seed.shape)} {seed.dtype} on {seed.device}")
        seed_value = 0
    else:
        seed_value, seed = (int(seed) + 2 ** 63) % 2 ** 64 - 2 ** 63, None  # modulo 2^64, as the kernel's 64 bits hold it
    if _use_kernels(x):
        return _DropoutFn.apply(x, residual, seed, seed_value, stream, threshold)
    number = seed_value if seed is None else int(seed)
    keep = _philox_numbers(number, stream, x.numel(), x.device).view(x.shape) >= threshold
    wide = torch.promote_types(x.dtype, torch.float32)
    y = torch.where(keep, x.to(wide) * (65536.0 / (65536 - threshold)), 0.0)
    if residual is not None:
        y = y + residual.to(wide)
    return y.to(x.dtype)
