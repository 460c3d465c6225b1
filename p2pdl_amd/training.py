"""The operators of a trainer's local step, on hand-written gfx950 kernels.

Between two rounds of the protocol a trainer runs the reference's ``train``
(training/train.py:7-22, called at node/node.py:322-324) and sends the change
of its model (``p2pdl_amd.node.local_update``).  This module has what such a
step computes for a model of a language model's build, each operator with its
gradient:

  layer_norm            normalisation of rows, weight and bias
  dropout               mask from a counter-based generator, never stored; adds a residual
  gated_linear          act(x w_gate^T) * (x w_up^T), a feed-forward block's first half
  linear_cross_entropy  loss of a linear head (no bias) over a large vocabulary, logits never kept

Every operator has a differentiable form (above) and a pair ``*_forward`` /
``*_backward`` that a hand-written or captured step calls directly.  Types:
float32, float16, bfloat16, one per call; sums and statistics are held in 32
bits.  Of 16-bit types the last two operators' gradients are rounded to the type
once, as operands of their products (small sizes keep them in 32 bits).  float32
products are float32 products (larger ones are sums over 16-bit parts: an
infinity among their operands may come out as NaN, operands below 2^-110 lose
digits).  No result depends on the order of atomics or on where a tensor lies, and
a dropout mask depends on (seed, offset) alone, so a step run again on the same
inputs gives the same bits, and a local update the same digest.

Tensors are [..., features]; rows may have a pitch (a slice of a wider
tensor is read in place), other layouts are copied.  Work is launched on the
current stream of the tensors' device; workspaces come from torch's
allocator, per call.  A differentiable form, and its backward pass, refuses to
be captured into a graph: torch accumulates the gradients of its leaves on the streams of
earlier backward passes, which a capture cannot join; a captured step calls
the ``*_forward`` / ``*_backward`` pairs.
"""
from __future__ import annotations

import ctypes

import torch
from torch.autograd.function import once_differentiable

from . import _native as N

# The calls of a step on dense tensors, checked and launched in C++ (csrc/train_host.cpp); its functions
# return None for what the Python below has to copy, widen or refuse.
_host = N.host_extension("_train_host")
_bound = False

DTYPES = {torch.float32: N.P2P_DTYPE_F32, torch.float16: N.P2P_DTYPE_F16, torch.bfloat16: N.P2P_DTYPE_BF16}
ACTIVATIONS = {"silu": N.P2P_ACT_SILU, "gelu": N.P2P_ACT_GELU, "relu": N.P2P_ACT_RELU}
MAX_NORM_COLS = 16384
MAX_FEATURES = (1 << 22) - 8  # of a product
MAX_UNITS = (1 << 21) - 8


def _bind() -> None:
    """Gives csrc/train_host.cpp the library's functions (those of struct Abi there, in that order)."""
    global _bound
    L = N.lib()
    names = ("layernorm_fwd", "layernorm_bwd_workspace", "layernorm_bwd", "dropout", "gated_linear_workspace",
             "gated_linear_fwd", "gated_linear_bwd", "linear_ce_workspace", "linear_ce_fwd", "linear_ce_bwd")
    _host.bind(tuple(ctypes.cast(getattr(L, "p2p_" + n), ctypes.c_void_p).value for n in names), N.check,
               torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream)
    _bound = True


def _call(fn, what: str, dev: torch.device, *args) -> None:
    """fn(*args, the current stream of dev) with dev as the current device."""
    if not _bound:
        _bind()
    if dev.index == torch._C._cuda_getDevice():
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(dev.index))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, N.stream_handle(dev))
    if rc:
        N.check(rc, what)


def _dtype(x: torch.Tensor, name: str) -> int:
    dt = DTYPES.get(x.dtype)
    if dt is None or not x.is_cuda or not x.numel():
        N.require_device(x)
        if dt is None:
            raise TypeError(f"{name}: expected float32, float16 or bfloat16, got {x.dtype}")
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError(f"{name}: needs a last dimension of at least one feature, got shape {tuple(x.shape)}")
    return dt


def _like(t: torch.Tensor, x: torch.Tensor, name: str, shape) -> None:
    if t.shape == shape and t.dtype is x.dtype and t.device == x.device:
        return
    if t.dtype != x.dtype:
        raise TypeError(f"{name}: expected {x.dtype}, got {t.dtype}")
    if t.device != x.device:
        raise RuntimeError(f"{name}: expected all tensors on {x.device}, got {t.device}")
    raise ValueError(f"{name}: expected shape {tuple(shape)}, got {tuple(t.shape)}")


def _new(x: torch.Tensor) -> torch.Tensor:
    """A dense tensor of x's shape and type."""
    return torch.empty_like(x) if x.is_contiguous() else torch.empty(x.shape, dtype=x.dtype, device=x.device)


def _pair(shape, dtype: torch.dtype, dev: torch.device):
    """Two tensors of their own (a view of a common one could not be changed in place once autograd returns it)."""
    return torch.empty(shape, dtype=dtype, device=dev), torch.empty(shape, dtype=dtype, device=dev)


def _stat(t: torch.Tensor, x: torch.Tensor, name: str, shape) -> None:
    """A dense float32 tensor that a forward pass left for its backward pass."""
    if t.shape == shape and t.dtype is torch.float32 and t.device == x.device and t.is_contiguous():
        return
    if t.dtype != torch.float32:
        raise TypeError(f"{name}: expected float32, got {t.dtype}")
    if t.device != x.device:
        raise RuntimeError(f"{name}: expected all tensors on {x.device}, got {t.device}")
    raise ValueError(f"{name}: expected a contiguous tensor of shape {tuple(shape)}, got {tuple(t.shape)}")


def _rows(t: torch.Tensor):
    """(tensor, row pitch): t itself where its rows are dense and evenly spaced, else a copy."""
    cols = t.shape[-1]
    if t.is_contiguous():
        return t, cols
    if t.dim() == 2 and t.stride(0) >= cols and (t.stride(1) == 1 or cols == 1):
        return t, t.stride(0)
    if t.dim() > 2:
        try:
            flat = t.view(-1, cols)
        except RuntimeError:
            return t.contiguous(), cols
        return _rows(flat)
    return t.contiguous(), cols


def _ptr(t):
    return None if t is None else t.data_ptr()


def _workspace(nbytes: int, dev: torch.device, what: str):
    if nbytes < 0:
        N.check(nbytes, what)
    return torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None


def _refuse_capture(what: str) -> None:
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"{what}: the differentiable form cannot be captured into a graph; "
                           f"call {what}_forward and {what}_backward")


def _no_capture(what: str, *tensors) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        _refuse_capture(what)


# ------------------------------------------------------------------ layer norm
def _norm_inputs(x, weight, bias):
    dt = _dtype(x, "x")
    if x.shape[-1] > MAX_NORM_COLS:
        raise ValueError(f"x: rows of at most {MAX_NORM_COLS} features, got {x.shape[-1]}")
    if bias is not None and weight is None:
        raise ValueError("bias: needs a weight")
    for t, name in ((weight, "weight"), (bias, "bias")):
        if t is not None:
            _like(t, x, name, x.shape[-1:])
    return dt


def layer_norm_forward(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
                       eps: float = 1e-5):
    """y = (x - mean) / sqrt(var + eps) * weight + bias over the last dimension
    (at most 16384 features).  Returns (y, mean, rstd), the latter two float32
    of x's leading shape, for layer_norm_backward."""
    done = _host.layer_norm_forward(x, weight, bias, eps)
    if done is not None:
        return done
    dt = _norm_inputs(x, weight, bias)
    dev, cols = x.device, x.shape[-1]
    rows = x.numel() // cols
    y = _new(x)
    mean, rstd = _pair(x.shape[:-1], torch.float32, dev)
    if rows:
        xr, ld = _rows(x)
        w = None if weight is None else weight.contiguous()
        b = None if bias is None else bias.contiguous()
        _call(N.lib().p2p_layernorm_fwd, "p2p_layernorm_fwd", dev, xr.data_ptr(), ld, _ptr(w), _ptr(b), rows, cols, eps,
              y.data_ptr(), mean.data_ptr(), rstd.data_ptr(), dt)
    return y, mean, rstd


def layer_norm_backward(dy: torch.Tensor, x: torch.Tensor, mean: torch.Tensor, rstd: torch.Tensor,
                        weight: torch.Tensor | None = None):
    """(dx, dweight, dbias) of layer_norm_forward; the latter two are None without a weight."""
    done = _host.layer_norm_backward(dy, x, mean, rstd, weight)
    if done is not None:
        return done
    dt = _norm_inputs(x, weight, None)
    _like(dy, x, "dy", x.shape)
    _stat(mean, x, "mean", x.shape[:-1])
    _stat(rstd, x, "rstd", x.shape[:-1])
    dev, cols = x.device, x.shape[-1]
    rows = x.numel() // cols
    dx = _new(x)
    dw = db = None
    if weight is not None:
        dw, db = _pair((cols,), x.dtype, dev)
    if rows:
        L = N.lib()
        xr, ldx = _rows(x)
        dyr, lddy = _rows(dy)
        w = ws = None
        nbytes = 0
        if weight is not None:
            w = weight.contiguous()
            nbytes = L.p2p_layernorm_bwd_workspace(rows, cols, dt)
            ws = _workspace(nbytes, dev, "p2p_layernorm_bwd_workspace")
        _call(L.p2p_layernorm_bwd, "p2p_layernorm_bwd", dev, dyr.data_ptr(), lddy, xr.data_ptr(), ldx, _ptr(w),
              mean.data_ptr(), rstd.data_ptr(), rows, cols, dx.data_ptr(), _ptr(dw), _ptr(db), _ptr(ws), nbytes, dt)
    elif weight is not None:
        dw.zero_()
        db.zero_()
    return dx, dw, db


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd = layer_norm_forward(x, weight, bias, eps)
        ctx.save_for_backward(x, weight, mean, rstd)
        ctx.has_bias = bias is not None
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        _refuse_capture("layer_norm")
        x, weight, mean, rstd = ctx.saved_tensors
        dx, dw, db = layer_norm_backward(dy, x, mean, rstd, weight)
        return dx, dw, db if ctx.has_bias else None, None


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-5) -> torch.Tensor:
    """Differentiable layer norm over the last dimension (layer_norm_forward's arguments)."""
    _no_capture("layer_norm", x, weight, bias)
    return _LayerNorm.apply(x, weight, bias, eps)


# ------------------------------------------------------------------ dropout
def _dropout(x, p, seed, offset, residual):
    done = _host.dropout(x, p, seed, offset, residual)
    if done is not None:
        return done
    dt = _dtype(x, "x")
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"p: expected a probability in [0, 1], got {p}")
    if not 0 <= seed < 1 << 64:
        raise ValueError(f"seed: expected an integer in [0, 2^64), got {seed}")
    offset_dev = None
    if isinstance(offset, torch.Tensor):
        if offset.dtype != torch.int64 or offset.numel() != 1 or offset.device != x.device:
            raise ValueError(f"offset: expected one int64 on {x.device}, got {offset.dtype} of {offset.numel()} elements "
                             f"on {offset.device}")
        offset, offset_dev = 0, offset
    elif not 0 <= offset < 1 << 64:
        raise ValueError(f"offset: expected an integer in [0, 2^64), got {offset}")
    if residual is not None:
        _like(residual, x, "residual", x.shape)
        residual = residual.contiguous()
    n = x.numel()
    y = _new(x)
    if n:
        xc = x.contiguous()
        _call(N.lib().p2p_dropout, "p2p_dropout", x.device, xc.data_ptr(), _ptr(residual), n, p, seed, offset,
              _ptr(offset_dev), y.data_ptr(), dt)
    return y


def dropout_blocks(numel: int) -> int:
    """How many counters a dropout of ``numel`` elements uses: the least distance of two
    offsets whose masks share no random number."""
    return -(-numel // 4)


def dropout_forward(x: torch.Tensor, p: float, seed: int, offset: int | torch.Tensor = 0,
                    residual: torch.Tensor | None = None) -> torch.Tensor:
    """x with each element dropped (set to 0) with probability p, the others
    divided by 1 - p, plus ``residual`` if given.

    Element i (in row-major order) is kept if word i % 4 of Philox4x32-10's
    block ``offset`` + i // 4 under the key ``seed`` is at least floor(p * 2^32): the
    mask is a function of (seed, offset) and is not stored.  ``offset`` may be a
    one-element int64 tensor on x's device, read when the kernel runs: a captured
    step advances it (by dropout_blocks) between replays."""
    return _dropout(x, p, seed, offset, residual)


def dropout_backward(dy: torch.Tensor, p: float, seed: int, offset: int | torch.Tensor = 0) -> torch.Tensor:
    """The gradient of x of dropout_forward with the same p, seed and offset (a residual's is dy)."""
    return _dropout(dy, p, seed, offset, None)


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, seed, offset, residual):
        # the mask is drawn again in the backward pass: a counter that moves on by then is kept as it is now
        ctx.at = (p, seed, offset.clone() if isinstance(offset, torch.Tensor) else offset)
        return _dropout(x, *ctx.at, residual)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        _refuse_capture("dropout")
        dx = dropout_backward(dy, *ctx.at) if ctx.needs_input_grad[0] else None
        return dx, None, None, None, dy if ctx.needs_input_grad[4] else None


def dropout(x: torch.Tensor, p: float, seed: int, offset: int | torch.Tensor = 0,
            residual: torch.Tensor | None = None) -> torch.Tensor:
    """Differentiable dropout (dropout_forward's arguments)."""
    _no_capture("dropout", x, residual)
    return _Dropout.apply(x, p, seed, offset, residual)


# ------------------------------------------------------------------ gated linear layer
def _gated_inputs(x, w_gate, w_up, activation):
    dt = _dtype(x, "x")
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"unknown activation {activation!r}; expected one of {sorted(ACTIVATIONS)}")
    if w_gate.dim() != 2 or w_gate.shape[0] == 0:
        raise ValueError(f"w_gate: expected a [units, features] weight, got shape {tuple(w_gate.shape)}")
    _like(w_gate, x, "w_gate", (w_gate.shape[0], x.shape[-1]))
    _like(w_up, x, "w_up", w_gate.shape)
    if x.shape[-1] > MAX_FEATURES or w_gate.shape[0] > MAX_UNITS:
        raise ValueError(f"at most {MAX_FEATURES} features and {MAX_UNITS} units, got {tuple(w_gate.shape)}")
    return dt, act


def _gated_args(x, w_gate, w_up, dt, act):
    """The call's struct, and the tensors that it points into."""
    a = N.GatedLinearArgs()
    xr, a.ldx = _rows(x)
    wg, a.ldg = _rows(w_gate)
    wu, a.ldu = _rows(w_up)
    a.x, a.w_gate, a.w_up = xr.data_ptr(), wg.data_ptr(), wu.data_ptr()
    a.hidden, a.units = x.shape[-1], w_gate.shape[0]
    a.tokens = x.numel() // x.shape[-1]
    a.activation, a.dtype = act, dt
    return a, (xr, wg, wu)


def gated_linear_forward(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, activation: str = "silu",
                         save: bool = True):
    """h = act(x w_gate^T) * (x w_up^T), x [..., features], weights [units,
    features], act "silu", "gelu" (exact) or "relu".  Returns (h, gate, up): the
    two products in float32, which gated_linear_backward reads (None with ``save``
    false, for inference)."""
    done = _host.gated_linear_forward(x, w_gate, w_up, ACTIVATIONS.get(activation), save)
    if done is not None:
        return done
    dt, act = _gated_inputs(x, w_gate, w_up, activation)
    dev, shape = x.device, x.shape[:-1] + w_gate.shape[:1]
    h = torch.empty(shape, dtype=x.dtype, device=dev)
    gate = up = None
    if save:
        gate, up = _pair(shape, torch.float32, dev)
    if x.numel():
        L = N.lib()
        a, keep = _gated_args(x, w_gate, w_up, dt, act)
        a.h, a.gate, a.up = h.data_ptr(), _ptr(gate), _ptr(up)
        nbytes = L.p2p_gated_linear_workspace(a, 0)
        ws = _workspace(nbytes, dev, "p2p_gated_linear_workspace")
        _call(L.p2p_gated_linear_fwd, "p2p_gated_linear_fwd", dev, a, _ptr(ws), nbytes)
        del keep
    return h, gate, up


def gated_linear_backward(dh: torch.Tensor, x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor,
                          gate: torch.Tensor, up: torch.Tensor, activation: str = "silu"):
    """(dx, dw_gate, dw_up) of gated_linear_forward."""
    done = _host.gated_linear_backward(dh, x, w_gate, w_up, gate, up, ACTIVATIONS.get(activation))
    if done is not None:
        return done
    dt, act = _gated_inputs(x, w_gate, w_up, activation)
    dev, shape = x.device, x.shape[:-1] + w_gate.shape[:1]
    _like(dh, x, "dh", shape)
    _stat(gate, x, "gate", shape)
    _stat(up, x, "up", shape)
    dx, dwg, dwu = _new(x), _new(w_gate), _new(w_up)
    if x.numel():
        L = N.lib()
        a, keep = _gated_args(x, w_gate, w_up, dt, act)
        dhr, a.lddh = _rows(dh)
        a.gate, a.up, a.dh = gate.data_ptr(), up.data_ptr(), dhr.data_ptr()
        a.dx, a.dw_gate, a.dw_up = dx.data_ptr(), dwg.data_ptr(), dwu.data_ptr()
        nbytes = L.p2p_gated_linear_workspace(a, 1)
        ws = _workspace(nbytes, dev, "p2p_gated_linear_workspace")
        _call(L.p2p_gated_linear_bwd, "p2p_gated_linear_bwd", dev, a, _ptr(ws), nbytes)
        del keep
    else:
        dwg.zero_()
        dwu.zero_()
    return dx, dwg, dwu


class _GatedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, activation):
        h, gate, up = gated_linear_forward(x, w_gate, w_up, activation, save=any(ctx.needs_input_grad))
        ctx.save_for_backward(x, w_gate, w_up, gate, up)
        ctx.activation = activation
        return h

    @staticmethod
    @once_differentiable
    def backward(ctx, dh):
        _refuse_capture("gated_linear")
        x, w_gate, w_up, gate, up = ctx.saved_tensors
        return gated_linear_backward(dh, x, w_gate, w_up, gate, up, ctx.activation) + (None,)


def gated_linear(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, activation: str = "silu") -> torch.Tensor:
    """Differentiable gated linear layer (gated_linear_forward's arguments)."""
    _no_capture("gated_linear", x, w_gate, w_up)
    return _GatedLinear.apply(x, w_gate, w_up, activation)


# ------------------------------------------------------------------ linear cross entropy
def _ce_args(x, weight, target, ignore_index):
    dt = _dtype(x, "x")
    if weight.dim() != 2 or weight.shape[0] == 0:
        raise ValueError(f"weight: expected a [vocabulary, features] weight, got shape {tuple(weight.shape)}")
    _like(weight, x, "weight", (weight.shape[0], x.shape[-1]))
    if target.dtype != torch.int64:
        raise TypeError(f"target: expected int64, got {target.dtype}")
    if target.device != x.device:
        raise RuntimeError(f"target: expected all tensors on {x.device}, got {target.device}")
    if target.shape != x.shape[:-1]:
        raise ValueError(f"target: expected shape {tuple(x.shape[:-1])}, got {tuple(target.shape)}")
    if x.shape[-1] > MAX_FEATURES:
        raise ValueError(f"at most {MAX_FEATURES} features, got {x.shape[-1]}")
    if not -(1 << 63) <= ignore_index < 1 << 63:
        raise ValueError(f"ignore_index: expected a 64-bit integer, got {ignore_index}")
    a = N.LinearCeArgs()
    xr, a.ldx = _rows(x)
    wr, a.ldw = _rows(weight)
    t = target.contiguous()
    a.x, a.w, a.target = xr.data_ptr(), wr.data_ptr(), t.data_ptr()
    a.hidden, a.vocab = x.shape[-1], weight.shape[0]
    a.tokens = x.numel() // x.shape[-1]
    a.ignore_index, a.dtype = ignore_index, dt
    return a, (xr, wr, t)


def linear_cross_entropy_forward(x: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, ignore_index: int = -100,
                                 reduction: str = "mean"):
    """Softmax cross entropy of the logits x weight^T against ``target``; neither
    pass keeps the logits (a small head's stand in its workspace during a call).  x
    [..., features], weight [vocabulary, features], target int64 of x's leading shape.  Tokens whose target is ``ignore_index`` do not count;
    ``reduction`` is "mean" over the others (0 where there are none) or "sum".  A
    target outside the vocabulary gives NaN.

    Returns (loss, lse, norm), float32: the loss (0-d), the log of each token's sum
    of exponentials and the factor of the mean, which the backward pass reads."""
    if reduction not in ("mean", "sum"):
        raise ValueError(f"unknown reduction {reduction!r}; expected 'mean' or 'sum'")
    done = _host.linear_cross_entropy_forward(x, weight, target, ignore_index, reduction == "mean")
    if done is not None:
        return done
    a, keep = _ce_args(x, weight, target, ignore_index)
    dev = x.device
    loss, norm = _pair((), torch.float32, dev)
    lse = torch.empty(target.shape, dtype=torch.float32, device=dev)
    a.mean = reduction == "mean"
    a.loss, a.lse, a.norm = loss.data_ptr(), lse.data_ptr(), norm.data_ptr()
    L = N.lib()
    nbytes = L.p2p_linear_ce_workspace(a, 0)
    ws = _workspace(nbytes, dev, "p2p_linear_ce_workspace")
    _call(L.p2p_linear_ce_fwd, "p2p_linear_ce_fwd", dev, a, _ptr(ws), nbytes)
    del keep
    return loss, lse, norm


def linear_cross_entropy_backward(x: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, lse: torch.Tensor,
                                  norm: torch.Tensor, dloss: torch.Tensor | None = None, ignore_index: int = -100):
    """(dx, dweight) of linear_cross_entropy_forward's loss, times ``dloss`` (one
    float32 on the device; a loss scale, say) if given."""
    done = _host.linear_cross_entropy_backward(x, weight, target, lse, norm, dloss, ignore_index)
    if done is not None:
        return done
    a, keep = _ce_args(x, weight, target, ignore_index)
    _stat(lse, x, "lse", target.shape)
    _stat(norm, x, "norm", torch.Size(()))
    dev = x.device
    if dloss is not None and (dloss.dtype != torch.float32 or dloss.numel() != 1 or dloss.device != dev):
        raise ValueError(f"dloss: expected one float32 on {dev}, got {dloss.dtype} of {dloss.numel()} elements on "
                         f"{dloss.device}")
    dx, dw = _new(x), _new(weight)
    if x.numel():
        a.lse, a.norm, a.dloss = lse.data_ptr(), norm.data_ptr(), _ptr(dloss)
        a.dx, a.dw = dx.data_ptr(), dw.data_ptr()
        L = N.lib()
        nbytes = L.p2p_linear_ce_workspace(a, 1)
        ws = _workspace(nbytes, dev, "p2p_linear_ce_workspace")
        _call(L.p2p_linear_ce_bwd, "p2p_linear_ce_bwd", dev, a, _ptr(ws), nbytes)
    else:
        dw.zero_()
    del keep
    return dx, dw


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, target, ignore_index, reduction):
        loss, lse, norm = linear_cross_entropy_forward(x, weight, target, ignore_index, reduction)
        ctx.save_for_backward(x, weight, target, lse, norm)
        ctx.ignore_index = ignore_index
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss):
        _refuse_capture("linear_cross_entropy")
        x, weight, target, lse, norm = ctx.saved_tensors
        return linear_cross_entropy_backward(x, weight, target, lse, norm, dloss, ctx.ignore_index) + (None, None, None)


def linear_cross_entropy(x: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, ignore_index: int = -100,
                         reduction: str = "mean") -> torch.Tensor:
    """Differentiable cross entropy of a linear head (linear_cross_entropy_forward's arguments)."""
    _no_capture("linear_cross_entropy", x, weight)
    return _LinearCrossEntropy.apply(x, weight, target, ignore_index, reduction)
