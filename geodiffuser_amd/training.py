"""What a program that learns needs of the text tower and the transformer blocks, on torch's autograd: the token embedding, the norms around a
block with its gate and residual, and clipping of the gradients.  The arithmetic is in the HIP kernels behind ``ops``; the same
functions serve no-grad passes.

The reference learns text embeddings and latents only (GeoDiffuser/utils/inversion.py:213-259, GeoDiffuser/utils/optimization.py:165-253) and
leaves these operators to torch."""
from __future__ import annotations

from typing import Iterable, Optional, Union

import torch

from . import ops
from .ops import Norm  # noqa: F401 - part of this module's interface


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
    device that nothing (a hook, a replaced ``forward``, autocast) makes into something else.  Norms that do not learn keep their path."""
    if not (torch.is_grad_enabled() and x.is_cuda and x.is_contiguous() and x.shape[-1] <= 16384 and x.numel() > 0
            and x.dtype in (torch.float16, torch.bfloat16, torch.float32) and not torch.is_autocast_enabled()):
        return False
    return (any(p.requires_grad for n in norms for p in n.parameters())
            and all(type(n) is torch.nn.LayerNorm and "forward" not in n.__dict__
                    and not (n._forward_hooks or n._forward_pre_hooks or n._backward_hooks or n._backward_pre_hooks) for n in norms)
            and all(p.dtype == x.dtype and p.device == x.device and p.is_contiguous() for n in norms for p in n.parameters()))


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
