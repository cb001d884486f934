"""Training operators of a Swin block, with their gradients.

The reference's patch runs eager torch in training (torch-ext/crumpet/monai_patch.py:137-151),
and so do the patched methods here unless :func:`enable_training_kernels` is called on a model.
The operators behind it, each usable by itself:

* :func:`relative_position_buckets` / :func:`relative_position_bias`: the learned
  relative-position bias ``table[index]`` per head and the gradient of its table;
* :func:`swin_window_attention_train`: window attention from the packed qkv with that bias and
  the shifted-window mask, differentiable in qkv and the table.  Nothing but its inputs is kept
  for the backward pass;
* :func:`norm_gate_residual`: post-norm, gate, per-sample residual scale, residual add and the
  next norm in one pass each way;
* :func:`gelu_checkpoint` / :func:`checkpointed_mlp`: GELU whose input is kept in 8 bits, and
  the MLP around it.

``*_backward`` functions are the gradients as plain calls, for programs that do without
autograd.  All run on the current CUDA stream and return without waiting for it; results do not
change from run to run (no atomics).  CUDA tensors only, as elsewhere in the package.
"""

from __future__ import annotations

import sys
import weakref
from typing import NamedTuple, Sequence

import torch
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from . import _ops as _native
from . import profiling as _prof
from .fused_attention import head_dim_supported

_DTYPES = (torch.float32, torch.float16, torch.bfloat16)
GROUP = 32  # neighbouring channels that share one scale of an 8-bit checkpoint
MAX_CHANNELS = 4096  # of norm_gate_residual
_ITEM = 512  # most pairs of one bucket that one warp sums (half of it where buckets are longer)


def _require_cuda(what: str, *tensors) -> None:
    for t in tensors:
        if t is not None and not t.is_cuda:
            raise RuntimeError(f"crumpet_b200 runs {what} on CUDA devices only (got {t.device})")


def _needs_grad(*tensors) -> bool:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


def _launch(name: str, work, *args):
    """One call of a training op of the library (which checks its arguments and allocates what it
    returns), counted, and timed while a timer is active; ``work`` gives its algorithmic work."""
    op = getattr(_native.require(), name)
    token = _prof.kernel_begin(name, work) if _prof._active else None
    res = op(*args)
    _prof.count(name)
    _prof.kernel_end(token)
    return res


def _nbytes(*tensors) -> int:
    return sum(t.numel() * t.element_size() for t in tensors if t is not None)


# ------------------------------------------------------------------ relative-position bias
class RelativePositionBuckets(NamedTuple):
    """A fixed bucket index ``[rows, cols]``, laid out once for the bias and its gradient
    (:func:`relative_position_buckets`)."""

    index: torch.Tensor  # int64 [rows, cols]
    pairs: torch.Tensor  # int32 [rows, cols]: the same
    order: torch.Tensor  # int32 [rows * cols]: the pairs sorted by bucket
    items: torch.Tensor  # int32 [n, 3]: bucket (-1: one of several items), begin, end
    multi: torch.Tensor  # int32 [m, 3]: bucket of several items, its first item, past its last
    num_buckets: int


def relative_position_buckets(index: torch.Tensor, num_buckets: int) -> RelativePositionBuckets:
    """Lay out ``index`` (integers ``[rows, cols]`` in ``[0, num_buckets)``, the bucket of every
    query / key pair) for :func:`relative_position_bias` and
    :func:`swin_window_attention_train`.  Made once for a module's index (for a window clamped
    to a smaller volume, of its slice ``index[:n, :n]``): it sorts the pairs and checks their
    values, which waits for the device; the plan is then ready for any stream."""
    if index.ndim != 2 or index.is_floating_point() or index.is_complex() or index.dtype == torch.bool:
        raise ValueError("index must be an integer tensor [rows, cols]")
    num_buckets = int(num_buckets)
    if num_buckets < 1:
        raise ValueError("num_buckets must be positive")
    if index.numel() >= 2 ** 31 or num_buckets >= 2 ** 31:
        raise ValueError("index must hold fewer than 2^31 pairs and buckets")
    # a copy: a later write to the caller's index does not reach a part of the plan
    index = torch.empty(index.shape, dtype=torch.int64, device=index.device).copy_(index.detach())
    flat = index.reshape(-1)
    if flat.numel() and (int(flat.min()) < 0 or int(flat.max()) >= num_buckets):
        raise ValueError(f"index values must lie in [0, {num_buckets})")
    order = torch.sort(flat, stable=True).indices
    count = torch.bincount(flat, minlength=num_buckets)
    begin = torch.cumsum(count, 0) - count
    # a 7x7x7 window's buckets (up to 343 pairs) are one item each, so nothing is to be joined;
    # long buckets are cut finer, for more warps
    size = _ITEM if int(count.max()) <= _ITEM else _ITEM // 2
    parts = torch.clamp((count + size - 1) // size, min=1)  # an empty bucket has one item too
    bucket = torch.repeat_interleave(torch.arange(num_buckets, device=index.device), parts)
    first = torch.cumsum(parts, 0) - parts
    part = torch.arange(bucket.numel(), device=index.device) - first[bucket]
    lo = begin[bucket] + part * size
    hi = torch.minimum(lo + size, (begin + count)[bucket])
    several = parts > 1
    items = torch.stack((torch.where(several[bucket], -1, bucket), lo, hi), 1)
    which = torch.nonzero(several).reshape(-1)
    multi = torch.stack((which, first[which], (first + parts)[which]), 1)
    plan = RelativePositionBuckets(index, index.int(), order.int(), items.int().contiguous(),
                                   multi.int().contiguous(), num_buckets)
    if index.is_cuda:  # kept for later calls, whatever their stream
        torch.cuda.current_stream(index.device).synchronize()
    return plan


def _check_table(table: torch.Tensor, buckets: RelativePositionBuckets) -> None:
    if table.ndim != 2 or table.shape[0] != buckets.num_buckets:
        raise ValueError(f"table must have shape [{buckets.num_buckets}, heads]")
    if table.dtype not in _DTYPES:
        raise TypeError("CRUMPET supports torch.float32, torch.float16 and torch.bfloat16")


def _bias_forward(table, buckets, dtype):
    pairs = buckets.pairs
    return _launch("relative_position_bias", lambda: {
        "bytes": pairs.numel() * (table.shape[1] * dtype.itemsize + 4)}, table, pairs, dtype)


class _Bias(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, buckets, dtype):
        ctx.buckets, ctx.dtype = buckets, table.dtype
        return _bias_forward(table, buckets, dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        return relative_position_bias_backward(grad, ctx.buckets, ctx.dtype), None, None


def relative_position_bias(table: torch.Tensor, buckets: RelativePositionBuckets,
                           dtype: torch.dtype | None = None) -> torch.Tensor:
    """``table[index].permute(2, 0, 1)`` as a contiguous ``[heads, rows, cols]`` in ``dtype``
    (default: the table's), differentiable in ``table [num_buckets, heads]``."""
    _check_table(table, buckets)
    dtype = table.dtype if dtype is None else dtype
    if dtype not in _DTYPES:
        raise TypeError("CRUMPET supports torch.float32, torch.float16 and torch.bfloat16")
    if table.device.type == "meta":
        return torch.empty((int(table.shape[1]), *buckets.pairs.shape), dtype=dtype, device="meta")
    _require_cuda("relative_position_bias", table, buckets.pairs)
    if _needs_grad(table):
        return _Bias.apply(table, buckets, dtype)
    return _bias_forward(table, buckets, dtype)


def relative_position_bias_backward(grad_bias: torch.Tensor, buckets: RelativePositionBuckets,
                                    dtype: torch.dtype | None = None) -> torch.Tensor:
    """Gradient of the table, ``[num_buckets, heads]`` in ``dtype`` (default: ``grad_bias``'s),
    from the gradient ``[heads, rows, cols]`` of the bias: per bucket the fp32 sum over its
    pairs, rounded once."""
    if grad_bias.ndim != 3 or grad_bias.shape[1:] != buckets.pairs.shape:
        raise ValueError(f"grad_bias must have shape [heads, {', '.join(map(str, buckets.pairs.shape))}]")
    dtype = grad_bias.dtype if dtype is None else dtype
    if grad_bias.dtype not in _DTYPES or dtype not in _DTYPES:
        raise TypeError("CRUMPET supports torch.float32, torch.float16 and torch.bfloat16")
    _require_cuda("relative_position_bias_backward", grad_bias, buckets.order)
    return _launch("relative_position_bias_backward", lambda: {
        "bytes": _nbytes(grad_bias, buckets.order)}, grad_bias, buckets.order, buckets.items,
        buckets.multi, buckets.num_buckets, dtype)


# ------------------------------------------------------------------------- window attention
def _place(qkv, table, buckets, num_windows, window_size, shift_size, scale):
    """The arguments as the ops take them (which check the rest)."""
    if qkv.ndim != 5:
        raise ValueError("qkv must have shape [B, N, 3, H, head_dim]")
    _check_table(table, buckets)
    _require_cuda("window attention", qkv, table, buckets.pairs)
    if window_size is None:
        window_size = (qkv.shape[1], 1, 1)
    if scale is None:
        scale = qkv.shape[4] ** -0.5
    return num_windows, window_size, shift_size, scale


def _attention_work(qkv, tensors: int, products: int):
    B, N, _, H, D = qkv.shape
    return {"bytes": tensors * B * H * N * D * qkv.element_size(),
            "flops": 2 * products * B * H * N * N * D, "exps": B * H * N * N}


def _attention_forward(qkv, table, buckets, place):
    return _launch("swin_window_attention_train", lambda: _attention_work(qkv, 4, 2), qkv, table,
                   buckets.index, buckets.pairs, *place)


def _attention_backward(grad_out, qkv, table, buckets, place):
    return _launch("swin_window_attention_backward", lambda: _attention_work(qkv, 7, 5), grad_out,
                   qkv, table, buckets.pairs, buckets.order, buckets.items, buckets.multi, *place)


class _WindowAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, qkv, table, buckets, place):
        ctx.save_for_backward(qkv, table)
        ctx.buckets, ctx.place = buckets, place
        return _attention_forward(qkv, table, buckets, place)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out):
        qkv, table = ctx.saved_tensors
        return (*_attention_backward(grad_out, qkv, table, ctx.buckets, ctx.place), None, None)


def swin_window_attention_train(
    qkv: torch.Tensor,
    table: torch.Tensor,
    buckets: RelativePositionBuckets,
    num_windows: Sequence[int] = (1, 1, 1),
    window_size: Sequence[int] | None = None,
    shift_size: Sequence[int] = (0, 0, 0),
    scale: float | None = None,
) -> torch.Tensor:
    """:func:`~crumpet_b200.swin_window_attention_qkv` for training: the same result (in
    fp32 to rounding, about 1e-6; in 16 bits the bias is rounded to them, which the gradient does
    not see), from ``qkv [B, N, 3, H, head_dim]``, the bias ``table
    [num_buckets, H]`` and its ``buckets`` (of the ``[N, N]`` index), differentiable in ``qkv`` and
    ``table``."""
    place = _place(qkv, table, buckets, num_windows, window_size, shift_size, scale)
    if _needs_grad(qkv, table):
        return _WindowAttention.apply(qkv, table, buckets, place)
    return _attention_forward(qkv, table, buckets, place)


def swin_window_attention_backward(
    grad_out: torch.Tensor,
    qkv: torch.Tensor,
    table: torch.Tensor,
    buckets: RelativePositionBuckets,
    num_windows: Sequence[int] = (1, 1, 1),
    window_size: Sequence[int] | None = None,
    shift_size: Sequence[int] = (0, 0, 0),
    scale: float | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """``(grad_qkv, grad_table)`` of :func:`swin_window_attention_train` from ``grad_out
    [B, N, H * head_dim]`` and the forward's own arguments, in the dtypes of ``qkv`` and
    ``table``."""
    place = _place(qkv, table, buckets, num_windows, window_size, shift_size, scale)
    _require_cuda("window attention", grad_out)
    return _attention_backward(grad_out, qkv, table, buckets, place)


# ------------------------------------------------- norms, gate and residual between branches
class NormGateGrads(NamedTuple):
    """Gradients of :func:`norm_gate_residual`; None where the argument was not given."""

    residual: torch.Tensor
    branch: torch.Tensor
    gate: torch.Tensor | None
    post_weight: torch.Tensor | None
    post_bias: torch.Tensor | None
    pre_weight: torch.Tensor | None
    pre_bias: torch.Tensor | None


def _pair(norm, name):
    if norm is None:
        return None, None
    if len(norm) != 2:
        raise ValueError(f"{name} must be a (weight, bias) pair")
    return norm


def _norm_gate_forward(branch, residual, gate, row_scale, post_w, post_b, pre_w, pre_b, eps):
    res = _launch("norm_gate_residual", lambda: {
        "bytes": _nbytes(branch, residual, residual, branch if pre_w is not None else None)},
        branch, residual, gate, row_scale, post_w, post_b, pre_w, pre_b, eps)
    return res if pre_w is not None else (res[0], None)


def _norm_gate_backward(grad_out, grad_normed, out, branch, gate, row_scale, post_w, post_b, pre_w,
                        eps):
    res = _launch("norm_gate_residual_backward", lambda: {
        "bytes": _nbytes(grad_out, grad_normed, out if pre_w is not None else None,
                         branch if gate is not None or post_w is not None else None, out, branch)},
        grad_out, grad_normed, out, branch, gate, row_scale, post_w, post_b, pre_w, eps)
    sums = iter(res[2:])
    return NormGateGrads(res[0], res[1], None if gate is None else next(sums),
                         *((None, None) if post_w is None else (next(sums), next(sums))),
                         *((None, None) if pre_w is None else (next(sums), next(sums))))


class _NormGate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, branch, residual, gate, row_scale, post_w, post_b, pre_w, pre_b, eps):
        out, normed = _norm_gate_forward(branch, residual, gate, row_scale, post_w, post_b, pre_w,
                                         pre_b, eps)
        # branch is read again for the gate's and the post-norm's gradients alone
        ctx.save_for_backward(branch if gate is not None or post_w is not None else None, out, gate,
                              row_scale, post_w, post_b, pre_w)
        ctx.eps, ctx.branch_dtype = eps, branch.dtype
        ctx.dtypes = tuple(None if t is None else t.dtype
                           for t in (gate, post_w, post_b, pre_w, pre_b))
        return out if normed is None else (out, normed)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out, grad_normed=None):
        branch, out, *params = ctx.saved_tensors
        if branch is None:  # not read: its shape and dtype, without the memory
            branch = out.new_empty((), dtype=ctx.branch_dtype).expand(out.shape)
        g = _norm_gate_backward(grad_out, grad_normed, out, branch, *params, ctx.eps)
        gate, *norms = (None if t is None else t.to(dt) for t, dt in zip(g[2:], ctx.dtypes))
        return g.branch, g.residual, gate, None, *norms, None


def norm_gate_residual(
    branch: torch.Tensor,
    residual: torch.Tensor,
    gate: torch.Tensor | None = None,
    row_scale: torch.Tensor | None = None,
    post_norm: tuple[torch.Tensor, torch.Tensor] | None = None,
    pre_norm: tuple[torch.Tensor, torch.Tensor] | None = None,
    eps: float = 1e-5,
) -> tuple[torch.Tensor, torch.Tensor | None]:
    """``(out, normed)`` of ``out = residual + row_scale * gate * post_norm(branch)`` and
    ``normed = pre_norm(out)``.

    ``branch [..., C]``; ``residual`` has its shape, in its dtype or float32 (the stream under
    autocast), and gives ``out``'s dtype; ``normed`` (None without ``pre_norm``) has the
    branch's.  ``post_norm`` / ``pre_norm`` are the (weight, bias) of a LayerNorm over C with
    ``eps``, ``gate [C]`` a layer scale, ``row_scale [samples]`` a factor per sample (drop path:
    0 or 1 / keep; the leading dimensions are cut evenly).  Differentiable in all but
    ``row_scale``.  C at most 4096.
    """
    post_w, post_b = _pair(post_norm, "post_norm")
    pre_w, pre_b = _pair(pre_norm, "pre_norm")
    if branch.device.type == "meta":
        return torch.empty_like(residual), None if pre_w is None else torch.empty_like(branch)
    _require_cuda("norm_gate_residual", branch, residual)
    if _needs_grad(branch, residual, gate, post_w, post_b, pre_w, pre_b):
        res = _NormGate.apply(branch, residual, gate, row_scale, post_w, post_b, pre_w, pre_b, eps)
        return res if pre_w is not None else (res, None)
    return _norm_gate_forward(branch, residual, gate, row_scale, post_w, post_b, pre_w, pre_b, eps)


def norm_gate_residual_backward(
    grad_out: torch.Tensor,
    grad_normed: torch.Tensor | None,
    out: torch.Tensor,
    branch: torch.Tensor,
    gate: torch.Tensor | None = None,
    row_scale: torch.Tensor | None = None,
    post_norm: tuple[torch.Tensor, torch.Tensor] | None = None,
    pre_norm: tuple[torch.Tensor, torch.Tensor] | None = None,
    eps: float = 1e-5,
) -> NormGateGrads:
    """Gradients of :func:`norm_gate_residual` from those of its results, its own ``out`` and
    the forward's arguments; ``grad_normed`` is None without ``pre_norm``.  The norms' and the
    gate's gradients are float32."""
    post_w, post_b = _pair(post_norm, "post_norm")
    pre_w, _ = _pair(pre_norm, "pre_norm")
    _require_cuda("norm_gate_residual", branch, out, grad_out, grad_normed)
    return _norm_gate_backward(grad_out, grad_normed, out, branch, gate, row_scale, post_w, post_b,
                               pre_w, eps)


# -------------------------------------------------------------- 8-bit activation checkpoints
class KeptActivation(NamedTuple):
    """An activation ``[..., C]`` in 8 bits: per 32 neighbouring channels one power of two
    ``2^(scales - 127)`` and int8 multiples of it, as finite as the activation (``scales`` 255:
    the group held an infinity or NaN and reads back as NaN)."""

    kept: torch.Tensor    # int8 [..., C]
    scales: torch.Tensor  # uint8 [..., ceil(C / 32)]
    dtype: torch.dtype


def gelu_checkpoint(x: torch.Tensor) -> tuple[torch.Tensor, KeptActivation]:
    """``gelu(x)`` (of the normal distribution, as ``torch.nn.GELU()``; off by at most 0.75e-7 |x|
    before rounding) and ``x`` in 8 bits for :func:`gelu_checkpoint_backward`.  Called outside autograd (:func:`checkpointed_mlp` is the
    differentiable form)."""
    if _needs_grad(x):
        raise RuntimeError("gelu_checkpoint is not differentiable by itself; use "
                           "checkpointed_mlp, or call it under torch.no_grad()")
    _require_cuda("gelu_checkpoint", x)
    y, kept, scales = _launch("gelu_checkpoint", lambda: {
        "bytes": x.numel() * (2 * x.element_size() + 1 + 1 / GROUP)}, x)
    return y, KeptActivation(kept, scales, x.dtype)


def gelu_checkpoint_backward(grad_y: torch.Tensor, kept: KeptActivation
                             ) -> tuple[torch.Tensor, torch.Tensor]:
    """``(grad_x, again)`` from the gradient of ``y``: with ``u`` the kept input, ``grad_y *
    gelu'(u)`` and ``gelu(u)``, the input of the next Linear's weight gradient."""
    if grad_y.dtype != kept.dtype:
        raise ValueError("grad_y must have the shape and dtype of the kept activation")
    _require_cuda("gelu_checkpoint_backward", grad_y)
    return _launch("gelu_checkpoint_backward", lambda: {
        "bytes": grad_y.numel() * (3 * grad_y.element_size() + 1 + 1 / GROUP)}, grad_y, kept.kept,
        kept.scales)


def restore_activation(kept: KeptActivation) -> torch.Tensor:
    """The kept activation in its own dtype."""
    _require_cuda("restore_activation", kept.kept)
    return _launch("restore_activation", lambda: {
        "bytes": kept.kept.numel() * (1 + kept.dtype.itemsize)}, kept.kept, kept.scales, kept.dtype)


class _Mlp(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w1, b1, w2, b2, dtype):
        xc, w1c, w2c = x.to(dtype), w1.to(dtype), w2.to(dtype)
        # outside autocast: the operands are already in the compute dtype
        with torch.autocast("cuda", enabled=False):
            u = F.linear(xc, w1c, None if b1 is None else b1.to(dtype))
            y, kept = gelu_checkpoint(u)
            out = F.linear(y, w2c, None if b2 is None else b2.to(dtype))
        ctx.save_for_backward(xc, w1c, w2c, kept.kept, kept.scales)
        ctx.dtypes = tuple(None if t is None else t.dtype for t in (x, w1, b1, w2, b2))
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        x, w1, w2, kept, scales = ctx.saved_tensors
        needs = ctx.needs_input_grad  # products of frozen weights are left out
        grads = [None] * 5
        with torch.autocast("cuda", enabled=False):
            rows = lambda t: t.reshape(-1, t.shape[-1])  # noqa: E731
            grad = grad.to(x.dtype)
            if any(needs[:4]):
                grad_u, y = gelu_checkpoint_backward(grad @ w2,
                                                     KeptActivation(kept, scales, x.dtype))
            if needs[0]:
                grads[0] = grad_u @ w1
            if needs[1]:
                grads[1] = rows(grad_u).t() @ rows(x)
            if needs[2]:
                grads[2] = rows(grad_u).sum(0)
            if needs[3]:
                grads[3] = rows(grad).t() @ rows(y)
            if needs[4]:
                grads[4] = rows(grad).sum(0)
        return (*(None if g is None else g.to(dt) for g, dt in zip(grads, ctx.dtypes)), None)


def checkpointed_mlp(x: torch.Tensor, weight1: torch.Tensor, bias1: torch.Tensor | None,
                     weight2: torch.Tensor, bias2: torch.Tensor | None) -> torch.Tensor:
    """``linear2(gelu(linear1(x)))`` that keeps its hidden activation in 8 bits (a byte and
    1/32 per element instead of the Linear's output and GELU's) for the backward pass.

    Computes in the autocast dtype under autocast, else in ``x``'s.  The forward result is the
    unquantised one; the gradients of ``x``, ``weight1``, ``bias1`` and ``weight2`` see the
    hidden activation as 8 bits keep it.
    """
    if weight1.ndim != 2 or weight2.ndim != 2 or int(weight1.shape[1]) != int(x.shape[-1]) \
            or int(weight2.shape[1]) != int(weight1.shape[0]):
        raise ValueError("weight1 must be [hidden, C] and weight2 [out, hidden]")
    _require_cuda("checkpointed_mlp", x, weight1, weight2)
    dtype = torch.get_autocast_dtype("cuda") if torch.is_autocast_enabled("cuda") else x.dtype
    if dtype not in _DTYPES:
        raise TypeError("CRUMPET supports torch.float32, torch.float16 and torch.bfloat16")
    return _Mlp.apply(x, weight1, bias1, weight2, bias2, dtype)


# ------------------------------------------------------------------- a Swin stage in training
# per attention module: its index, the index's version, and {n: buckets}
_buckets = weakref.WeakKeyDictionary()


def _module_buckets(attn, n: int) -> RelativePositionBuckets:
    """The buckets of the module's own index for windows of n tokens, laid out on first use and
    again if the index tensor is replaced or written to."""
    index = attn.relative_position_index
    kept = _buckets.get(attn)
    if kept is None or kept[0] is not index or kept[1] != index._version:
        kept = _buckets[attn] = (index, index._version, {})
    if n not in kept[2]:
        kept[2][n] = relative_position_buckets(index[:n, :n],
                                               attn.relative_position_bias_table.shape[0])
    return kept[2][n]


def _off(module) -> bool:
    """Whether a dropout-like module (or None) does nothing."""
    return module is None or isinstance(module, torch.nn.Identity) \
        or getattr(module, "p", None) == 0.0


def _plain(module, kind) -> bool:
    """Exactly a ``kind`` with the class's own forward: not a subclass (adapters,
    parametrizations), not an instance whose forward was replaced."""
    return type(module) is kind and "forward" not in module.__dict__


def _hooked(module) -> bool:
    return bool(module._forward_hooks or module._forward_pre_hooks or module._backward_hooks
                or module._backward_pre_hooks)


def _fits(norm, C: int) -> bool:
    return (_plain(norm, torch.nn.LayerNorm) and tuple(norm.normalized_shape) == (C,)
            and norm.weight is not None and norm.bias is not None and norm.eps > 0)


def _known(blk) -> bool:
    """Whether the block, its attention and its MLP are the Swin classes of its own module."""
    swin = sys.modules[type(blk).__module__]
    mlp = getattr(swin, "Mlp", getattr(swin, "MLPBlock", None))
    return (_plain(blk, getattr(swin, "SwinTransformerBlock", None))
            and _plain(blk.attn, getattr(swin, "WindowAttention", None)) and _plain(blk.mlp, mlp))


def _block_trains(blk, C: int) -> bool:
    """Whether the training kernels compute exactly what the block does.  They call the block's
    qkv and proj as modules and read the parameters of all others, so those have to be the plain
    classes, and nothing may be hooked to them."""
    if not _known(blk):
        return False
    attn, mlp = blk.attn, blk.mlp
    path = getattr(blk, "drop_path", None)
    softmax = getattr(attn, "softmax", None)
    heads = int(attn.num_heads)
    passed_by = (blk, blk.norm1, blk.norm2, path, attn, softmax, attn.attn_drop, attn.proj_drop, mlp,
                 mlp.linear1, mlp.linear2, mlp.fn, getattr(mlp, "drop1", None),
                 getattr(mlp, "drop2", None))
    return (C <= MAX_CHANNELS and _fits(blk.norm1, C) and _fits(blk.norm2, C)
            and C % heads == 0 and head_dim_supported(C // heads)
            and (softmax is None or _plain(softmax, torch.nn.Softmax) and softmax.dim == -1)
            and _off(attn.attn_drop) and _off(attn.proj_drop)
            and _plain(mlp.linear1, torch.nn.Linear) and _plain(mlp.linear2, torch.nn.Linear)
            and _plain(mlp.fn, torch.nn.GELU) and mlp.fn.approximate == "none"
            and _off(getattr(mlp, "drop1", None)) and _off(getattr(mlp, "drop2", None))
            and (_off(path) or (type(path).__name__ == "DropPath" and hasattr(path, "drop_prob")
                                and "forward" not in path.__dict__
                                and getattr(path, "scale_by_keep", True)))
            and not getattr(blk, "use_checkpoint", False)
            and not torch.nn.modules.module._has_any_global_hook()
            and not any(m is not None and _hooked(m) for m in passed_by))


def _path_scale(blk, samples: int, device) -> torch.Tensor | None:
    """Drop path's factor per sample: 0, or 1 / keep with probability keep; None where it is not
    in training mode."""
    path = getattr(blk, "drop_path", None)
    drop = float(getattr(path, "drop_prob", 0.0) or 0.0)
    if drop == 0.0 or not path.training:
        return None
    keep = 1.0 - drop
    kept = torch.rand(samples, device=device) < keep
    return kept.float() / keep if keep > 0 else kept.float()


def _train_branch(blk, normed, window_size, shift_size):
    """The attention branch of a block from norm1's output: pad, roll + partition, qkv, window
    attention, proj, back."""
    from . import fused_shift_partition_3d, fused_unshift_unpartition_3d

    attn = blk.attn
    b, d, h, w, c = normed.shape
    pad = [-s % ws for s, ws in zip((d, h, w), window_size)]
    if any(pad):
        normed = F.pad(normed, (0, 0, 0, pad[2], 0, pad[1], 0, pad[0]))
    dims = tuple(int(s) for s in normed.shape[1:4])
    windows = fused_shift_partition_3d(normed, window_size, shift_size)
    n, heads = int(windows.shape[1]), int(attn.num_heads)
    qkv = attn.qkv(windows).view(windows.shape[0], n, 3, heads, c // heads)
    num_windows = tuple(s // ws for s, ws in zip(dims, window_size))
    out = swin_window_attention_train(qkv, attn.relative_position_bias_table,
                                      _module_buckets(attn, n), num_windows, window_size,
                                      shift_size, attn.scale)
    out = attn.proj(out)
    x = fused_unshift_unpartition_3d(out, b, *dims, c, window_size, shift_size)
    return x[:, :d, :h, :w].contiguous() if any(pad) else x


def _train_layer(layer, x, get_window_size):
    """A Swin stage (channels-first in and out) on the training operators: between two branches
    one :func:`norm_gate_residual` adds the residual and takes the next norm."""
    b, c, d, h, w = (int(s) for s in x.shape)
    x = x.permute(0, 2, 3, 4, 1).contiguous()
    blocks = list(layer.blocks)
    compute = torch.get_autocast_dtype("cuda") if torch.is_autocast_enabled("cuda") else x.dtype
    normed = blocks[0].norm1(x).to(compute)
    for i, blk in enumerate(blocks):
        window_size, shift_size = get_window_size((d, h, w), blk.window_size, blk.shift_size)
        window_size, shift_size = tuple(map(int, window_size)), tuple(map(int, shift_size))
        branch = _train_branch(blk, normed, window_size, shift_size)
        x, normed = norm_gate_residual(
            branch, x, row_scale=_path_scale(blk, b, x.device),
            pre_norm=(blk.norm2.weight, blk.norm2.bias), eps=blk.norm2.eps)
        mlp = blk.mlp
        if layer.__dict__.get(_EIGHT_BITS, True):
            branch = checkpointed_mlp(normed, mlp.linear1.weight, mlp.linear1.bias,
                                      mlp.linear2.weight, mlp.linear2.bias)
        else:
            branch = mlp(normed)
        after = blocks[i + 1].norm1 if i + 1 < len(blocks) else None
        x, normed = norm_gate_residual(
            branch, x, row_scale=_path_scale(blk, b, x.device),
            pre_norm=None if after is None else (after.weight, after.bias),
            eps=blk.norm2.eps if after is None else after.eps)
    if layer.downsample is not None:
        x = layer.downsample(x)
    return x.permute(0, 4, 1, 2, 3).contiguous()


_EIGHT_BITS = "_crumpet_eight_bits"  # of a switched stage: keep hidden activations in 8 bits


def _stage_trains(layer, x) -> bool:
    return (x.dim() == 5 and x.is_cuda and layer.training and x.dtype in _DTYPES
            and all(_block_trains(blk, int(x.shape[1])) for blk in layer.blocks))


def _layer_forward(layer, x):
    base = type(layer)._crumpet_stage
    if not _stage_trains(layer, x):
        return base.forward(layer, x)
    if torch.is_autocast_enabled("cuda") and x.dtype not in (torch.float32,
                                                            torch.get_autocast_dtype("cuda")):
        x = x.float()
    return _train_layer(layer, x, sys.modules[base.__module__].get_window_size)


# A switched stage is an instance of a subclass of its class.  Its forward is then the copy's own
# in every copy of the module (nn.DataParallel's replicas, deepcopy, pickles), which a method kept
# in the instance is not.
_switched: dict = {}


def _restore_stage(base):
    layer = base.__new__(base)
    layer.__class__ = _switched_class(base)
    return layer


def _switched_class(base):
    """The subclass of stage class ``base`` on the training kernels."""
    cls = _switched.get(base)
    if cls is None:
        cls = _switched[base] = type(base.__name__, (base,), {
            "__module__": base.__module__, "__qualname__": base.__qualname__,
            "__doc__": base.__doc__, "_crumpet_stage": base, "forward": _layer_forward,
            # pickled as the class it is made from (its own has no name to be found by)
            "__reduce_ex__": lambda self, protocol: (_restore_stage, (base,), self.__getstate__()),
        })
    return cls


def _is_switched(module) -> bool:
    return _switched.get(getattr(type(module), "_crumpet_stage", None)) is type(module)


def _layers(model):
    return [m for m in model.modules()
            if hasattr(m, "blocks") and hasattr(m, "downsample") and hasattr(m, "window_size")
            and hasattr(sys.modules[type(m).__module__], "get_window_size")]


def enable_training_kernels(model: torch.nn.Module, eight_bit_activations: bool = True) -> int:
    """Run the Swin stages (``BasicLayer`` of MONAI or of ``crumpet_b200.swin_unetr``) of
    ``model`` on the training operators while they are in training mode, on CUDA; returns how
    many.  A stage with what they do not compute (attention, projection or MLP dropout,
    activation checkpointing, another activation or norm, and in place of a block, its norms, its
    MLP or the MLP's Linears anything but the plain class: adapters, parametrizations, pruning,
    hooks) keeps its own forward, and so does eval mode.  Copies of the
    model (replicas, deepcopy, pickles) keep the switch; a file of a pickled model then needs this
    package to load.

    With ``eight_bit_activations`` the MLPs keep their hidden activation in 8 bits for the backward
    pass (:func:`checkpointed_mlp`), in fp32 training too: their gradients are then off by about 2^-8
    in the norm.  Without, the MLPs run as modules, at the memory and precision of eager ones.  Undone by :func:`disable_training_kernels`."""
    layers = [m for m in _layers(model) if "forward" not in m.__dict__]
    for layer in layers:
        if not _is_switched(layer):
            layer.__class__ = _switched_class(type(layer))
        layer.__dict__[_EIGHT_BITS] = bool(eight_bit_activations)
    return len(layers)


def disable_training_kernels(model: torch.nn.Module) -> int:
    """Undo :func:`enable_training_kernels`; returns how many stages it changed back."""
    layers = [m for m in model.modules() if _is_switched(m)]
    for layer in layers:
        layer.__class__ = type(layer)._crumpet_stage
        layer.__dict__.pop(_EIGHT_BITS, None)
    return len(layers)


def _fake_norm_gate_backward(grad_out, grad_normed, out, branch, gate, row_scale, post_w, post_b,
                             pre_w, eps):
    n = (gate is not None) + 2 * (post_w is not None) + 2 * (pre_w is not None)
    vector = branch.new_empty(branch.shape[-1:], dtype=torch.float32)
    return [out.new_empty(out.shape), branch.new_empty(branch.shape),
            *(torch.empty_like(vector) for _ in range(n))]


# What the ops that return new tensors return, for tracing (shape and dtype only)
FAKE_IMPLS = {
    "relative_position_bias": lambda table, pairs, dtype: table.new_empty(
        (table.shape[1], *pairs.shape), dtype=dtype),
    "relative_position_bias_backward": lambda grad, order, items, multi, buckets, dtype:
        grad.new_empty((buckets, grad.shape[0]), dtype=dtype),
    "swin_window_attention_train": lambda qkv, table, index, pairs, nw, ws, ss, scale: qkv.new_empty(
        (qkv.shape[0], qkv.shape[1], qkv.shape[3] * qkv.shape[4])),
    "swin_window_attention_backward": lambda grad, qkv, table, pairs, order, items, multi, nw, ws,
        ss, scale: (qkv.new_empty(qkv.shape), table.new_empty(table.shape)),
    "norm_gate_residual": lambda branch, residual, gate, scale, post_w, post_b, pre_w, pre_b, eps:
        [residual.new_empty(residual.shape)]
        + ([] if pre_w is None else [branch.new_empty(branch.shape)]),
    "norm_gate_residual_backward": _fake_norm_gate_backward,
    "gelu_checkpoint": lambda x: (
        x.new_empty(x.shape), x.new_empty(x.shape, dtype=torch.int8),
        x.new_empty((*x.shape[:-1], -(-x.shape[-1] // GROUP)), dtype=torch.uint8)),
    "gelu_checkpoint_backward": lambda grad, kept, scales: (grad.new_empty(grad.shape),
                                                            grad.new_empty(grad.shape)),
    "restore_activation": lambda kept, scales, dtype: kept.new_empty(kept.shape, dtype=dtype),
}

__all__ = [
    "RelativePositionBuckets", "relative_position_buckets", "relative_position_bias",
    "relative_position_bias_backward", "swin_window_attention_train",
    "swin_window_attention_backward", "NormGateGrads", "norm_gate_residual",
    "norm_gate_residual_backward", "KeptActivation", "gelu_checkpoint",
    "gelu_checkpoint_backward", "restore_activation", "checkpointed_mlp",
    "enable_training_kernels", "disable_training_kernels",
]
