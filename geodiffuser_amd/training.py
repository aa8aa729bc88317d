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


class _EmbedFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, table, pos, scale, padding_idx):
        ctx.save_for_backward(ids)
        ctx.cfg = (table.shape[0], None if pos is None else pos.shape[0], scale, padding_idx)
        return ops.embed_tokens(ids, table, pos, scale)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        (ids,) = ctx.saved_tensors
        vocab, pos_rows, scale, padding_idx = ctx.cfg
        dy = dy.contiguous()
        return (None, ops.embed_tokens_bwd(ids, dy, vocab, scale, padding_idx) if ctx.needs_input_grad[1] else None,
                ops.embed_positions_bwd(dy, pos_rows) if ctx.needs_input_grad[2] else None, None, None)


def embed_tokens(ids, table, pos=None, scale: float = 1.0, padding_idx: Optional[int] = None):
    """``ops.embed_tokens`` with gradients for table and pos; row ``padding_idx`` of the table gets none."""
    return _EmbedFn.apply(ids, table, pos, scale, padding_idx)


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
    @torch.autograd.function.once_differentiable
    def backward(ctx, gs, gy):
        x, res, gate, pre_gamma, pre_beta, post_gamma, post_beta, stats = ctx.saved_tensors
        pre, post, res_scale = ctx.cfg
        names = ("dx", "dres", "dgate", "dpre_gamma", "dpre_beta", "dpost_gamma", "dpost_beta")
        if gs is None and gy is None:
            return (None,) * 10
        d = ops.block_norm_bwd(x, res, None if gy is None else gy.contiguous(), None if gs is None else gs.contiguous(), stats,
                               None if pre is None else Norm(pre[0], pre_gamma, pre_beta, pre[1]),
                               None if post is None else Norm(post[0], post_gamma, post_beta, post[1]), gate, res_scale,
                               need=[n for n, want in zip(names, ctx.needs_input_grad) if want])
        return tuple(d[n] for n in names) + (None, None, None)


def block_norm(x, res, pre: Optional[Norm], post: Optional[Norm] = None, gate=None, res_scale: float = 1.0):
    """``ops.block_norm`` -> (s, y) with gradients for x, res, gate and the norms' gamma / beta."""
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


def clip_grad_norm_(parameters: Union[torch.Tensor, Iterable[torch.Tensor]], max_norm: float, norm_type: float = 2.0):
    """torch.nn.utils.clip_grad_norm_ on ``ops.clip_grad_norm``: scales the parameters' gradients in place so that their joint norm is at most
    ``max_norm`` -> the norm before (0-d tensor on the device, nothing is synchronised; 0 if no parameter has a gradient)."""
    params = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    grads = [p.grad for p in params if p.grad is not None]
    if not grads:
        return torch.zeros(())
    return ops.clip_grad_norm([g.detach() for g in grads], max_norm, norm_type)
