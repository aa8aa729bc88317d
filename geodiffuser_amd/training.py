"""What a program that learns needs of the text tower and the transformer blocks, on torch's autograd: the token embedding, the norms around a
block with its gate and residual, and clipping of the gradients.  The arithmetic is in the HIP kernels behind ``ops``; the same
functions serve no-grad passes.

The reference learns text embeddings and latents only (GeoDiffuser/utils/inversion.py:213-259, GeoDiffuser/utils/optimization.py:165-253) and
leaves these operators to torch."""
from __future__ import annotations

from typing import Iterable, Optional, Union

import torch
from torch.autograd import forward_ad
from torch.nn.modules import module as _module

from . import ops
from .ops import Norm  # noqa: F401 - part of this module's interface

_PLAIN_TYPES = (torch.Tensor, torch.nn.Parameter)


def in_plain_torch(*tensors: torch.Tensor) -> bool:
    """Whether these are ordinary tensors of an ordinary eager pass, which is what a kernel that is handed addresses can serve.  Where not - under
    torch.func.grad / vmap / jvp, forward-mode differentiation, a dispatch mode (fake tensors, make_fx, counters), a jit or compiler trace,
    for tensor subclasses - the framework's modules keep to torch's own operations."""
    if (torch.compiler.is_compiling() or torch._C._len_torch_dispatch_stack() or torch._C._functorch.peek_interpreter_stack() is not None
            or forward_ad._current_level >= 0 or torch._C._get_tracing_state() is not None):
        return False
    return all(type(t) in _PLAIN_TYPES and not torch._C._functorch.is_legacy_batchedtensor(t) for t in tensors)


def is_stock(module: torch.nn.Module, kind: type) -> bool:
    """Whether calling the module runs kind.forward and nothing else: no subclass, replaced ``forward``, or hook of its own or of all modules."""
    return (type(module) is kind and "forward" not in module.__dict__ and not _module._has_any_global_hook()
            and not (module._forward_hooks or module._forward_pre_hooks or module._backward_hooks or module._backward_pre_hooks))


def _embed_grads_in_torch(ids, dy, vocab, pos_rows, scale, padding_idx):
    """The gradients of table and pos (None without position rows) as torch operations, in 32 bits or more, rounded once."""
    wide, L, C = torch.promote_types(dy.dtype, torch.float32), dy.shape[-2], dy.shape[-1]
    ok = (ids >= 0) & (ids < vocab)
    if padding_idx is not None:
        ok = ok & (ids != padding_idx)
    rows = torch.where(ok[..., None], dy.to(wide) * scale, 0.0)
    table = torch.ops.aten.embedding_dense_backward(rows, torch.where(ok, ids, 0), vocab, -1, False).to(dy.dtype) if vocab else dy.new_zeros(0, C)
    pos = None if pos_rows is None else torch.nn.functional.pad(dy.to(wide).sum_to_size(L, C), (0, 0, 0, pos_rows - L)).to(dy.dtype)
    return table, pos


class _EmbedFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, table, pos, scale, padding_idx):
        ctx.save_for_backward(ids)
        ctx.cfg = (table.shape[0], None if pos is None else pos.shape[0], scale, padding_idx)
        return ops.embed_tokens(ids, table, pos, scale)

    @staticmethod
    def backward(ctx, dy):
        (ids,) = ctx.saved_tensors
        vocab, pos_rows, scale, padding_idx = ctx.cfg
        if torch.is_grad_enabled() or not in_plain_torch(dy):            # create_graph, is_grads_batched
            table, pos = _embed_grads_in_torch(ids, dy, vocab, pos_rows, scale, padding_idx)
            return None, table if ctx.needs_input_grad[1] else None, pos if ctx.needs_input_grad[2] else None, None, None
        dy = dy.contiguous()
        return (None, ops.embed_tokens_bwd(ids, dy, vocab, scale, padding_idx) if ctx.needs_input_grad[1] else None,
                ops.embed_positions_bwd(dy, pos_rows) if ctx.needs_input_grad[2] else None, None, None)


def embed_tokens(ids, table, pos=None, scale: float = 1.0, padding_idx: Optional[int] = None):
    """``ops.embed_tokens`` with gradients for table and pos; row ``padding_idx`` of the table gets none.  Gradients that are themselves
    differentiated (create_graph) or batched (is_grads_batched) are computed by torch's operations."""
    return _EmbedFn.apply(ids, table, pos, scale, padding_idx)


def _norm_rows(v, kind, eps):
    """-> normalised rows, 1 / deviation"""
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    r = torch.rsqrt((v * v).mean(-1, keepdim=True) + eps)
    return v * r, r


def _norm_rows_grad(g, xh, r, kind):
    d = g - xh * (g * xh).mean(-1, keepdim=True)
    return r * (d - g.mean(-1, keepdim=True) if kind == "layer" else d)


def _block_norm_grads_in_torch(x, res, gy, gs, pre, post, gate, res_scale):
    """What ``ops.block_norm_bwd`` returns, as torch operations, in 32 bits or more, rounded once; differentiable w.r.t. every tensor."""
    wide, C, dtype = torch.promote_types(x.dtype, torch.float32), x.shape[-1], x.dtype
    up = lambda t: None if t is None else t.to(wide)
    X, G = up(x), up(gate)
    if G is not None and G.dim() == 2 and x.dim() >= 2:
        G = G.reshape(G.shape[0], *([1] * (x.dim() - 2)), C)
    scaled = lambda t, gamma: t if gamma is None else t * up(gamma)
    out = {}
    h = X
    if post is not None:
        xh, xr = _norm_rows(X, post.kind, post.eps)
        h = scaled(xh, post.gamma)
        if post.beta is not None:
            h = h + up(post.beta)
    ds = up(gs)
    if gy is not None:
        s = h if G is None else G * h
        sh, sr = _norm_rows(s if res is None else s + res_scale * up(res), pre.kind, pre.eps)
        ds = _norm_rows_grad(scaled(up(gy), pre.gamma), sh, sr, pre.kind)
        if gs is not None:
            ds = ds + up(gs)
    if pre is not None:
        none = torch.zeros(C, dtype=dtype, device=x.device)
        out["dpre_gamma"] = none if gy is None else (up(gy) * sh).sum_to_size(C)
        out["dpre_beta"] = none if gy is None else up(gy).sum_to_size(C)
    out["dres"] = res_scale * ds
    if G is not None:
        out["dgate"] = (ds * h).sum_to_size(G.shape).reshape(gate.shape)
        ds = G * ds
    if post is not None:
        out["dpost_gamma"], out["dpost_beta"] = (ds * xh).sum_to_size(C), ds.sum_to_size(C)
        ds = _norm_rows_grad(scaled(ds, post.gamma), xh, xr, post.kind)
    out["dx"] = ds
    return {k: v.to(dtype) for k, v in out.items()}


class _BlockNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, res, gate, pre_gamma, pre_beta, post_gamma, post_beta, pre, post, res_scale):
        pre_n = None if pre is None else Norm(pre[0], pre_gamma, pre_beta, pre[1])
        post_n = None if post is None else Norm(post[0], post_gamma, post_beta, post[1])
        s, y, stats = ops.block_norm(x, res, pre_n, post_n, gate, res_scale)
        ctx.save_for_backward(x, res, gate, pre_gamma, pre_beta, post_gamma, post_beta, stats)
        ctx.cfg = (pre, post, res_scale)
        ctx.set_materialize_grads(False)
        return (s.view_as(s) if s is x else s), y

    @staticmethod
    def backward(ctx, gs, gy):
        x, res, gate, pre_gamma, pre_beta, post_gamma, post_beta, stats = ctx.saved_tensors
        pre, post, res_scale = ctx.cfg
        names = ("dx", "dres", "dgate", "dpre_gamma", "dpre_beta", "dpost_gamma", "dpost_beta")
        if gs is None and gy is None:
            return (None,) * 10
        need = [n for n, want in zip(names, ctx.needs_input_grad) if want]
        pre = None if pre is None else Norm(pre[0], pre_gamma, pre_beta, pre[1])
        post = None if post is None else Norm(post[0], post_gamma, post_beta, post[1])
        if torch.is_grad_enabled() or not in_plain_torch(*(g for g in (gs, gy) if g is not None)):       # create_graph, is_grads_batched
            d = _block_norm_grads_in_torch(x, res, gy, gs, pre, post, gate, res_scale)
            return tuple(d[n] if n in need else None for n in names) + (None, None, None)
        d = ops.block_norm_bwd(x, res, None if gy is None else gy.contiguous(), None if gs is None else gs.contiguous(), stats, pre, post, gate, res_scale, need=need)
        return tuple(d[n] for n in names) + (None, None, None)


def block_norm(x, res, pre: Optional[Norm], post: Optional[Norm] = None, gate=None, res_scale: float = 1.0):
    """``ops.block_norm`` -> (s, y) with gradients for x, res, gate and the norms' gamma / beta.  Gradients that are themselves differentiated
    (create_graph) or batched (is_grads_batched) are computed by torch's operations."""
    return _BlockNormFn.apply(x, res, gate, pre and pre.gamma, pre and pre.beta, post and post.gamma, post and post.beta,
                              pre and (pre.kind, pre.eps), post and (post.kind, post.eps), res_scale)


def fuses_norms(x, norms) -> bool:
    """Whether a pass over x differentiates w.r.t. the weights of these norms and ``block_norm`` takes them: affine nn.LayerNorms of x's dtype and
    device that nothing (a hook, a replaced ``forward``, autocast, a transform) makes into something else.  Norms that do not learn keep
    their path."""
    if not in_plain_torch(x):
        return False
    if not (torch.is_grad_enabled() and x.is_cuda and x.is_contiguous() and x.shape[-1] <= 16384 and x.numel() > 0
            and x.dtype in (torch.float16, torch.bfloat16, torch.float32) and not torch.is_autocast_enabled()):
        return False
    return (any(p.requires_grad for n in norms for p in n.parameters())
            and all(is_stock(n, torch.nn.LayerNorm) for n in norms)
            and all(in_plain_torch(p) and p.dtype == x.dtype and p.device == x.device and p.is_contiguous() for n in norms for p in n.parameters()))


def layer_norm_of(module: torch.nn.LayerNorm) -> Norm:
    return Norm("layer", module.weight, module.bias, module.eps)


def _as_it_lies(grad):
    """A dense gradient's elements in the order of memory, whatever the order of its axes (a transposed parameter's gradient is transposed too):
    norm and scaling do not ask for more."""
    grad = grad.detach()
    if grad.is_contiguous() or not torch.ops.aten.is_non_overlapping_and_dense(grad):
        return grad
    return grad.as_strided((grad.numel(),), (1,))


def clip_grad_norm_(parameters: Union[torch.Tensor, Iterable[torch.Tensor]], max_norm: float, norm_type: float = 2.0):
    """torch.nn.utils.clip_grad_norm_ on ``ops.clip_grad_norm``: scales the parameters' gradients in place so that their joint norm is at most
    ``max_norm`` -> the norm before (0-d tensor on the device, nothing is synchronised; 0 if no parameter has a gradient).

    Gradients: f16 / bf16 / f32, mixed as they come, dense in any order of their axes, all on one GPU; ``norm_type`` 2 or inf.  A parameter
    listed twice is refused (torch counts and scales its gradient twice)."""
    params = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    grads = [p.grad for p in params if p.grad is not None]
    if not grads:
        return torch.zeros((), device=params[0].device if params else None)
    return ops.clip_grad_norm([_as_it_lies(g) for g in grads], max_norm, norm_type)
