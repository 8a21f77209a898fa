"""The tail of a training step: the loss of a linear head over many classes without its logits (``linear_ce_loss``) and the
orthogonalised update of an optimizer step (``newton_schulz``; ``optim.FusedMuon`` applies it).  Both run their products on the
matrix pipe through one core (csrc/nt_product.h).  ``fedicra_amd.ops`` re-exports them beside ``ce_loss`` and the other operators.

No CPU fallback: everything routes through fedicra_amd._lib."""
from __future__ import annotations

import contextlib

import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from . import _lib as L

NS_COEFFS = (3.4445, -4.7750, 2.0315)


_HERE = contextlib.nullcontext()


def _on(device):
    """The device's context where it is not the current one (entering it costs as much as a launch)."""
    return _HERE if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def newton_schulz(updates, steps=5, coeffs=NS_COEFFS, eps=1e-7):
    """The orthogonalised form of an update, by Newton-Schulz products:  X = U / (|U|_F + eps), then ``steps`` times
    X <- (a I + b A + c A A) X with A = X X^T (on the shorter side), i.e. the polynomial a s + b s^3 + c s^5 on every singular value.

    ``updates``: a matrix [m, n], a batch [B, m, n], or a list / tuple of matrices of any sizes -- all of a list's matrices share
    every kernel launch, so a model's filters are passed together.  fp32, bf16 or fp16, each result in its matrix's own type and shape;
    the products are accurate to 22 bits whatever that type is.  ``coeffs``: (a, b, c), or one triple per step.  A zero matrix gives
    zeros.  The result carries no gradient."""
    if isinstance(updates, torch.Tensor):
        if updates.dim() not in (2, 3):
            raise ValueError(f"newton_schulz: a matrix, a batch of matrices or a list of matrices, not {tuple(updates.shape)}")
        out = torch.empty(updates.shape, dtype=updates.dtype, device=updates.device)
        if updates.dim() == 2:
            _newton_schulz_into([updates], [out], steps, coeffs, eps)
        elif updates.shape[0]:
            _newton_schulz_into(list(updates.unbind(0)), list(out.unbind(0)), steps, coeffs, eps)
        return out
    updates = list(updates)
    if any(not isinstance(u, torch.Tensor) or u.dim() != 2 for u in updates):
        raise ValueError("newton_schulz: every entry of a list has to be a matrix")
    outs = [torch.empty(u.shape, dtype=u.dtype, device=u.device) for u in updates]
    if updates:
        _newton_schulz_into(updates, outs, steps, coeffs, eps)
    return outs


def _newton_schulz_into(updates, outs, steps, coeffs, eps):
    steps = int(steps)
    if steps < 1:
        raise ValueError("newton_schulz: steps must be at least 1")
    coeffs = tuple(coeffs)
    if len(coeffs) == 3 and not hasattr(coeffs[0], "__len__"):
        coeffs = (coeffs,) * steps
    if len(coeffs) != steps or any(len(c) != 3 for c in coeffs):
        raise ValueError("newton_schulz: coeffs is one triple (a, b, c), or one per step")
    if not eps >= 0.0:
        raise ValueError("newton_schulz: eps must not be negative")
    dev = updates[0].device
    if any(u.device != dev for u in updates):
        raise ValueError("newton_schulz: all matrices of a call live on one device")
    if any(u.numel() == 0 for u in updates):
        raise ValueError("newton_schulz: empty matrix")
    L._dev(updates[0])
    updates = [u.detach().contiguous() for u in updates]
    with _on(dev):
        L.newton_schulz(updates, outs, steps, coeffs, eps)


def _grad_slot(param, shape):
    """Where a gradient of `param` goes: (tensor to write, add to it?, what autograd gets).  A dense fp32 slice of the flat gradient buffer
    is added to in place (ops._grad_target), anything else gets a fresh tensor."""
    sink = getattr(param, "_fi_gview", None)
    if sink is not None:
        from . import ops
        tgt, _, ret = ops._grad_target(param)
        if ret is None and tgt.reshape(shape).data_ptr() == tgt.data_ptr():
            return tgt.reshape(shape), True, None
        if ret is not None and ret.reshape(shape).data_ptr() == ret.data_ptr():
            return ret.reshape(shape), True, ret
    g = param.new_empty(shape)
    return g, False, g if param.dim() == len(shape) else g.reshape(param.shape)


def _dense_rows(t, rows, cols):
    """[rows, cols] with dense rows that lie apart (a view; a copy where there is none: features apart, an expanded or overlapping tensor, rows so
    far apart that a tile's offsets would not fit)."""
    if t.dim() != 2:
        t = t.reshape(rows, cols)
    step, along = t.stride()
    return t if (along == 1 or cols == 1) and (rows == 1 or cols <= step <= 1 << 22) else t.contiguous()


def _fp32_row(t):
    return t if t is None or t.dtype == torch.float32 and t.is_contiguous() else t.detach().float().contiguous()


class _LinearCE(Function):
    @staticmethod
    def forward(ctx, x, weight, bias, labels, ignore_index, reduction):
        V, D = weight.shape[:2]
        T = labels.numel()
        x2, w2 = _dense_rows(x, T, D), _dense_rows(weight, V, D)
        b2, l2 = _fp32_row(bias), labels.contiguous()
        loss = torch.empty(labels.shape if reduction == "none" else (), dtype=torch.float32, device=x.device)
        with _on(x.device):
            desc = L.linear_ce_desc(x2, w2, l2, ignore_index, reduction)
            saved = L.linear_ce_fwd(desc, x2, w2, b2, l2, loss)
        ctx.save_for_backward(x, weight, bias, labels, saved)
        ctx.ignore_index, ctx.reduction = ignore_index, reduction
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        x, weight, bias, labels, saved = ctx.saved_tensors
        V, D = weight.shape[:2]
        x2, w2 = _dense_rows(x, labels.numel(), D), _dense_rows(weight, V, D)
        b2, l2 = _fp32_row(bias), labels.contiguous()
        gl = _fp32_row(g)
        dx = dw = db = gw = gb = None
        dw_add = db_add = False
        if ctx.needs_input_grad[0]:
            dx = x.new_empty(x.shape)
        if ctx.needs_input_grad[1]:
            dw, dw_add, gw = _grad_slot(weight, (V, D))
        if bias is not None and ctx.needs_input_grad[2]:
            if bias.dtype == torch.float32:
                db, db_add, gb = _grad_slot(bias, (V,))
            else:
                db = torch.empty(V, dtype=torch.float32, device=x.device)
        with _on(x.device):
            desc = L.linear_ce_desc(x2, w2, l2, ctx.ignore_index, ctx.reduction)    # (a hook on saved tensors may have moved the rows together)
            L.linear_ce_bwd(desc, x2, w2, b2, l2, saved, gl, dx, dw, dw_add, db, db_add)
        if db is not None and bias.dtype != torch.float32:
            gb = db.to(bias.dtype)
        return dx, gw, gb, None, None, None


def linear_ce_loss(x, weight, bias, labels, ignore_index=-100, reduction="mean"):
    """Softmax cross entropy of a linear head, ``CrossEntropyLoss(ignore_index)(x @ weight.T + bias, labels)``, without its logits: the
    product runs a tile at a time and its gradient a piece of rows x classes at a time.  Of rows x classes there are in memory pieces of at most 3 GiB and, above 128
    features or in fp32, 1/32 byte each (a row's statistics per 256 classes, the bias gradient's per 128 or 256 rows).

    x [..., D] fp32, bf16 or fp16 (any leading sizes; the labels' sizes); weight [V, D], or a 1x1 convolution's [V, D, 1, 1(, 1)], in x's type or
    fp32 (a 16-bit x then meets it rounded to x's type, like every operator here); bias [V] or None; labels int64, int32 or uint8.
    Rows whose label is ``ignore_index`` take no part, whatever x holds there, and cost (next to) nothing.  ``reduction``: "mean" over the
    labelled rows (NaN when there are none, as ``ce_loss``), "sum", or "none" -- a loss per row, 0 where ignored.  A label that is neither a class
    nor ``ignore_index`` makes the loss and the gradients NaN.  Classes may be ruled out by a bias of -inf or any large negative value.

    fp32: what fp32 products and sums give, whatever the sizes of rows, classes and features (from 1e-33 on).  16-bit x: logits and sums in fp32, the logits' gradient rounded
    once to fp16 (not at all up to 2^28 multiply-adds of fp16) relative to the row's own upstream gradient for dx, to the largest of all for the weight's: what
    lies below 2^-39 of that is lost, and so are bf16 values below 2^-39 of their tensor's largest.

    The gradients have the types of x, weight and bias (a parameter of a flat-store model: added to its slice of the flat buffer).  Twice
    differentiating is refused."""
    if reduction not in L.REDUCTIONS:
        raise ValueError(f"linear_ce_loss: reduction is 'mean', 'sum' or 'none', not {reduction!r}")
    if x.dim() < 1 or weight.dim() < 2 or x.shape[-1] != weight.shape[1] or weight.numel() != weight.shape[0] * weight.shape[1]:
        raise ValueError(f"linear_ce_loss: x [..., D] and weight [V, D] do not go together: {tuple(x.shape)}, {tuple(weight.shape)}")
    if labels.shape != x.shape[:-1]:
        raise ValueError(f"linear_ce_loss: labels {tuple(labels.shape)} for rows {tuple(x.shape[:-1])}")
    if bias is not None and bias.shape != weight.shape[:1]:
        raise ValueError(f"linear_ce_loss: bias {tuple(bias.shape)} for {weight.shape[0]} classes")
    if x.numel() == 0 or weight.numel() == 0:
        raise ValueError("linear_ce_loss: no rows, no classes or no features")
    if labels.dtype not in L.LABEL_TYPES:
        raise L.FiError(f"linear_ce_loss: labels are int64, int32 or uint8, not {labels.dtype}")
    if L.dt(weight.dtype) != L.dt(x.dtype) and weight.dtype != torch.float32:
        raise L.FiError(f"linear_ce_loss: weight is of x's type or fp32, not {weight.dtype} for {x.dtype}")
    dev = L._dev(x).device
    for t in (weight, labels) if bias is None else (weight, labels, bias):
        if L._dev(t).device != dev:
            raise ValueError("linear_ce_loss: x, weight, bias and labels live on one device")
    return _LinearCE.apply(x, weight, bias, labels, int(ignore_index), reduction)
