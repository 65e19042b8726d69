"""8-bit operators on the GPU (libp2n_hip.so): products in 8-bit integers with a scale for every token and channel, and
activation checkpoints in 8 bits for the backward pass.

The reference computes and keeps everything in float32 (reference src/models/point2net.py:9-34, train.py:124-131); these are
additions with a definition of their own.  The 8-bit rule they share: a set of values v has the scale
s = float32(max|v| / 127) and the codes q = clamp(round_half_even(v / s), -127, 127), the quotient taken exactly; s = 0 gives
q = 0; a NaN or an infinity among the v makes s NaN, and with it every result that the scale enters.

  quantize_tokens   codes and scales of the rows of a tensor
  Int8Weight        a weight matrix (and bias) put into 8 bits once, laid out for the matrix cores
  int8_linear       y = x W^T + b over rows of float32 or bfloat16, from one token to many
  int8_mlp          the layers of a shared MLP over (B, C, L), activations on chip; `SharedMLP.precision = "int8"` runs it
  act8_linear       W relu(norm(x)) + b (or W x + b) over (B, C, L), differentiable, its input kept in 8 bits
  act8_norm_relu    relu(norm(x)), differentiable, its input kept in 8 bits
                    `SharedMLP.checkpoint = "int8"` trains on these two

All functions take GPU tensors only and queue their work on the current stream of the tensors' device; nothing synchronises.
"""
import ctypes
from functools import lru_cache
from typing import Optional, Sequence

import torch
import torch.nn as nn

from . import _lib
from . import runtime as _rt


def _gpu(t: torch.Tensor, name: str, dtypes) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a GPU tensor")
    if t.dtype not in dtypes:
        raise TypeError(f"{name} must be {' or '.join(str(d).replace('torch.', '') for d in dtypes)}, got {t.dtype}")
    return t


def _no_grad_wanted(what: str, t: torch.Tensor) -> None:
    if t.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{what} has no backward pass (rounding to 8 bits has no gradient): call it under torch.no_grad()")


def _call(fn, what: str, dev: torch.device, *args) -> None:
    """fn(*args, current stream of dev) with dev as the current device, its return code turned into an error"""
    if torch._C._cuda_getDevice() == dev.index:
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(dev.index))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(dev.index))
    if rc:
        _lib.check(rc, what)


_TOKEN_TYPES = (torch.float32, torch.bfloat16)


def _rows(x: torch.Tensor):
    """(..., K) -> T, K, row stride and a tensor whose memory holds those rows"""
    shape = x.shape
    if not shape:
        raise ValueError("x must have at least one dimension")
    K = shape[-1]
    if K < 1:
        raise ValueError(f"x must have at least one value in a token, got {tuple(shape)}")
    if len(shape) == 2:
        ld, step = x.stride()
        if step == 1 and ld >= K:
            return shape[0], K, ld, x
    return x.numel() // K, K, K, x.contiguous()


@lru_cache(maxsize=256)
def _linear_bytes(T: int, K: int, N: int) -> int:
    """size of int8_linear's workspace (a number of the shape alone)"""
    return _lib.lib().p2n_int8_linear_workspace_bytes(T, K, N)


def quantize_tokens(x: torch.Tensor):
    """x (..., K) float32 or bfloat16 -> codes (..., K) int8, scale (...) float32: one scale for each row of K values."""
    _gpu(x, "x", _TOKEN_TYPES)
    _no_grad_wanted("quantize_tokens", x)
    T, K, ld, rows = _rows(x)
    codes = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    scale = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    _call(_lib.lib().p2n_quantize_tokens, "p2n_quantize_tokens", x.device, rows.data_ptr(), int(x.dtype == torch.bfloat16), T, K, ld,
          codes.data_ptr(), scale.data_ptr())
    return codes, scale


class Int8Weight:
    """A weight (N, K) -- or the (N, K, 1) of a Conv1d(kernel_size=1) -- and an optional bias (N), put into 8 bits with one scale
    per output channel and laid out for the kernels.  norm: a BatchNorm1d behind the product, folded in as eval mode applies it
    (running statistics).  Made once from the float32 values of that moment; make a new one after they changed."""

    def __init__(self, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, norm: Optional[nn.BatchNorm1d] = None):
        weight = _gpu(weight, "weight", (torch.float32,)).detach()
        if weight.dim() == 3 and weight.size(2) == 1:
            weight = weight.squeeze(2)
        if weight.dim() != 2:
            raise ValueError(f"weight must be (N,K) or (N,K,1), got {tuple(weight.shape)}")
        self.out_features, self.in_features = weight.shape
        self.device = weight.device
        if bias is not None:
            bias = _gpu(bias, "bias", (torch.float32,)).detach()
            if bias.shape != (self.out_features,) or bias.device != weight.device:
                raise ValueError(f"bias must be ({self.out_features},) on {weight.device}, got {tuple(bias.shape)} on {bias.device}")
            bias = bias.contiguous()
        fold = (None, None, None, None)
        if norm is not None:
            if not norm.affine or norm.running_mean is None:
                raise NotImplementedError("only a BatchNorm1d with affine=True and track_running_stats=True folds into the weight")
            if norm.num_features != self.out_features:
                raise ValueError(f"norm has {norm.num_features} channels, the weight {self.out_features}")
            fold = tuple(_gpu(t, "norm", (torch.float32,)).detach().contiguous() for t in (norm.weight, norm.bias, norm.running_mean, norm.running_var))
            if any(t.device != weight.device for t in fold):
                raise ValueError(f"norm must be on {weight.device}")
        L = _lib.lib()
        n = L.p2n_int8_weight_bytes(self.in_features, self.out_features)
        if n < 0:
            raise ValueError(f"weight (N,K) = {tuple(weight.shape)}: both must be in 1..65536")
        weight = weight.contiguous()
        self.image = torch.empty(n, dtype=torch.uint8, device=weight.device)
        _call(L.p2n_int8_pack_weight, "p2n_int8_pack_weight", weight.device, weight.data_ptr(), _rt.ptr(bias), self.in_features,
              self.out_features, *(_rt.ptr(t) for t in fold), 0.0 if norm is None else norm.eps, self.image.data_ptr())

    @property
    def scale(self) -> torch.Tensor:
        """(N,) float32, one for each output channel"""
        n = (self.out_features + 31) // 32 * 32
        return self.image[-8 * n:].view(torch.float32)[:self.out_features]

    @property
    def codes(self) -> torch.Tensor:
        """(N, K) int8, put back in order (a copy)"""
        ct, kt = (self.out_features + 31) // 32, (self.in_features + 63) // 64 * 2
        f = self.image[:ct * kt * 1024].view(torch.int8).view(ct, kt, 2, 32, 4, 4)     # tile, tile, half, row, group, j
        return f.permute(0, 3, 1, 4, 2, 5).reshape(ct * 32, kt * 32)[:self.out_features, :self.in_features].contiguous()


def int8_linear(x: torch.Tensor, weight: Int8Weight, relu: bool = False) -> torch.Tensor:
    """x (..., K) float32 or bfloat16 -> (..., N) of the same type: every token's values and the weight in 8 bits, their
    product exact in 32-bit integers, scaled, plus the weight's bias, then ReLU if asked."""
    _gpu(x, "x", _TOKEN_TYPES)
    _no_grad_wanted("int8_linear", x)
    T, K, ld, rows = _rows(x)
    if K != weight.in_features:
        raise ValueError(f"x has {K} values in a token, the weight takes {weight.in_features}")
    dev = x.device
    if dev != weight.device:
        raise ValueError(f"x is on {dev}, the weight on {weight.device}")
    N = weight.out_features
    y = x.new_empty((*x.shape[:-1], N))
    if T == 0:
        return y
    # from torch's allocator and not from the stream's shared buffer: a captured graph keeps the memory it was captured with
    nws = _linear_bytes(T, K, N)
    ws = torch.empty(nws, dtype=torch.uint8, device=dev) if nws else None
    _call(_lib.lib().p2n_int8_linear, "p2n_int8_linear", dev, rows.data_ptr(), int(x.dtype == torch.bfloat16), T, K, ld,
          weight.image.data_ptr(), N, int(relu), y.data_ptr(), _rt.ptr(ws), nws)
    return y


@lru_cache(maxsize=32)
def _arrays(layers: int):
    """C types of the widths and the images of so many layers"""
    return ctypes.c_int * (layers + 1), ctypes.c_void_p * layers


def int8_mlp(x: torch.Tensor, weights: Sequence[Int8Weight], last_relu: bool = True, group: int = 0) -> torch.Tensor:
    """x (B, C, L) float32 -> (B, N, L): the products of `weights` one after another over the columns of x, ReLU between them
    (and behind the last if last_relu); what passes from a layer to the next is put into 8 bits again, one scale a column.
    Such a hidden value is ((sum * token's scale) * channel's scale) + bias, each step rounded to float32, in that order: one step in it can
    move a code.
    group > 0: followed by the maximum over groups of `group` consecutive columns -> (B, N, L // group).
    1..8 layers, C <= 1024, every layer's N <= 256."""
    x = _gpu(x, "x", (torch.float32,))
    _no_grad_wanted("int8_mlp", x)
    if x.dim() != 3:
        raise ValueError(f"x must be (B,C,L), got {tuple(x.shape)}")
    weights = list(weights)
    if not weights:
        raise ValueError("int8_mlp needs at least one layer")
    B, C, L = x.shape
    dims, dev = [C], x.device
    for i, w in enumerate(weights):
        if w.in_features != dims[-1]:
            raise ValueError(f"layer {i} takes {w.in_features} channels, gets {dims[-1]}")
        if w.device != dev:
            raise ValueError(f"x is on {dev}, the weight of layer {i} on {w.device}")
        dims.append(w.out_features)
    if group < 0 or (group and L % group):
        raise ValueError(f"columns per cloud ({L}) are not a multiple of the group size ({group})")
    x = x.contiguous()
    lib = _lib.lib()
    # in the kernel: groups of 16 or 32; larger multiples of 32 finish on the maxima of 32, other sizes on the columns
    inner = 0 if group <= 1 else group if group == 16 else 32 if group % 32 == 0 else 0
    out = x.new_empty((B, dims[-1], L // inner if inner else L))
    ints, pointers = _arrays(len(weights))
    _call(lib.p2n_int8_mlp, "p2n_int8_mlp", dev, x.data_ptr(), B, L, len(weights), ints(*dims), pointers(*[w.image.data_ptr() for w in weights]),
          int(last_relu), inner, out.data_ptr())
    rest = group // inner if inner else group
    if rest > 1:
        res = x.new_empty((B, dims[-1], L // group))
        _call(lib.p2n_max_of_columns, "p2n_max_of_columns", dev, out.data_ptr(), res.numel(), rest, res.data_ptr())
        out = res
    return out


# ------------------------------------------------------------------ activation checkpoints in 8 bits
def _norm_args(norm: Optional[nn.BatchNorm1d], x: torch.Tensor, training: Optional[bool] = None):
    """gamma, beta, running mean, running variance, batches tracked (where it counts), momentum (< 0: running statistics used as they
    are), eps of a BatchNorm1d; `training` in place of its own flag"""
    if norm is None:
        return None, None, None, None, None, 0.0, 0.0
    if not isinstance(norm, nn.BatchNorm1d):
        raise TypeError(f"norm must be a BatchNorm1d or None, got {type(norm).__name__}")
    # straight from the module's dictionaries: its attribute access costs as much as a launch
    par, buf = norm._parameters, norm._buffers
    try:
        gamma, beta, mean, var = par["weight"], par["bias"], buf["running_mean"], buf["running_var"]
    except KeyError:                                     # parametrised: the values of the moment
        gamma, beta, mean, var = norm.weight, norm.bias, norm.running_mean, norm.running_var
    if gamma is None:
        raise NotImplementedError("the 8-bit checkpoint layers need BatchNorm1d(affine=True)")
    if gamma.size(0) != x.size(1):
        raise ValueError(f"norm has {gamma.size(0)} channels, x has {x.size(1)}")
    for t, name in ((gamma, "weight"), (beta, "bias"), (mean, "running_mean"), (var, "running_var")):
        if t is not None and not (t.dtype == torch.float32 and t.device == x.device and t.is_contiguous()):
            raise ValueError(f"norm.{name} must be a contiguous float32 tensor on the input's GPU")
    tracked = mean is not None
    if training is None:
        training = norm.training
    if training or not tracked:
        if x.size(0) * x.size(2) < 2:
            raise ValueError(f"Expected more than 1 value per channel when training, got input size {tuple(x.shape)}")
        if not training or not tracked:
            return gamma, beta, None, None, None, 0.0, norm.eps
        if norm.momentum is None:
            raise NotImplementedError("BatchNorm1d(momentum=None) (cumulative average) is not implemented on the GPU path")
        if not 0.0 <= norm.momentum <= 1.0:              # the kernels take a negative one as "running statistics as they are"
            raise ValueError(f"norm.momentum must be in [0,1], got {norm.momentum}")
        batches = buf["num_batches_tracked"]
        if batches is not None and not (batches.dtype == torch.int64 and batches.device == x.device):
            raise ValueError("norm.num_batches_tracked must be an int64 tensor on the input's GPU")
        return gamma, beta, mean, var, batches, norm.momentum, norm.eps
    return gamma, beta, mean, var, None, -1.0, norm.eps


def _bytes(n: int, device) -> torch.Tensor:
    return torch.empty(n, dtype=torch.uint8, device=device)


@lru_cache(maxsize=256)
def _act8_bytes(what: str, B: int, C: int, L: int, norm: bool, N: int):
    """sizes of the kept buffer and of the workspace (numbers of the shape alone)"""
    L_ = _lib.lib()
    nkept, nws = L_.p2n_act8_kept_bytes(B, C, L, int(norm)), L_.p2n_act8_workspace_bytes(B, C, L, N)
    if nkept == 0 or nws == 0:
        raise ValueError(f"{what}: " + L_.p2n_last_error().decode(errors="replace"))
    return nkept, nws


def _changed(mean, var, batches, momentum: float) -> None:
    """the kernels wrote these buffers through their addresses: autograd, and what is kept by a buffer's version, has to know"""
    if mean is not None and momentum >= 0:
        torch.autograd.graph.increment_version((mean, var) if batches is None else (mean, var, batches))


@torch.autograd.function.once_differentiable
def _once(function, ctx, g):
    """under create_graph: gradients that refuse to be differentiated (the decorator costs a launch's time, so it is taken only there)"""
    return function.gradients(ctx, g)


class _Act8Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, gamma, beta, running_mean, running_var, batches, momentum, eps):
        L_ = _lib.lib()
        B, K, L = x.shape
        N = weight.size(0)
        dev = x.device
        normed = gamma is not None
        nkept, nws = _act8_bytes("act8_linear", B, K, L, normed, N)
        kept, ws = _bytes(nkept, dev), _bytes(nws, dev)
        h = torch.empty((B, N, L), dtype=torch.float32, device=dev)
        _call(L_.p2n_act8_forward, "p2n_act8_forward", dev, x.data_ptr(), B, K, L, weight.data_ptr(), _rt.ptr(bias), N, _rt.ptr(gamma),
              _rt.ptr(beta), _rt.ptr(running_mean), _rt.ptr(running_var), _rt.ptr(batches), momentum, eps, h.data_ptr(), kept.data_ptr(), nkept,
              ws.data_ptr(), nws)
        _changed(running_mean, running_var, batches, momentum)
        ctx.save_for_backward(kept, weight, gamma, beta)
        ctx.meta = (B, K, L, N, normed and momentum < 0, bias is not None)
        return h

    @staticmethod
    def backward(ctx, g):
        return _once(_Act8Linear, ctx, g) if torch.is_grad_enabled() else _Act8Linear.gradients(ctx, g)

    @staticmethod
    def gradients(ctx, g):
        kept, weight, gamma, beta = ctx.saved_tensors
        B, K, L, N, frozen, has_bias = ctx.meta
        L_ = _lib.lib()
        g = g.contiguous()
        dev = g.device
        need = ctx.needs_input_grad
        normed = gamma is not None

        dgamma, dbeta = torch.empty_like(gamma) if normed and need[3] else None, torch.empty_like(beta) if normed and need[4] else None
        # the norm's gradients are formed on dx's way
        dx = torch.empty((B, K, L), dtype=torch.float32, device=dev) if need[0] or dgamma is not None or dbeta is not None else None
        dW = torch.empty_like(weight) if need[1] else None
        db = torch.empty(N, dtype=torch.float32, device=dev) if has_bias and need[2] else None
        nkept, nws = _act8_bytes("act8_linear", B, K, L, normed, N)
        ws = _bytes(nws, dev)
        _call(L_.p2n_act8_backward, "p2n_act8_backward", dev, g.data_ptr(), B, K, L, weight.data_ptr(), N, _rt.ptr(gamma), _rt.ptr(beta),
              int(frozen), kept.data_ptr(), nkept, _rt.ptr(dx), _rt.ptr(dW), _rt.ptr(db), _rt.ptr(dgamma), _rt.ptr(dbeta),
              ws.data_ptr(), nws)
        return dx if need[0] else None, dW, db, dgamma, dbeta, None, None, None, None, None


def act8_linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
                norm: Optional[nn.BatchNorm1d] = None, training: Optional[bool] = None) -> torch.Tensor:
    """x (B, K, L) float32 -> W relu(norm(x)) + b, or W x + b without a norm: (B, N, L), differentiable in x, weight (N, K) or
    (N, K, 1), bias and the norm's parameters.  The output is computed from the float32 values (finite ones: an infinity in a product's
    operands gives NaN); for the backward pass the
    normalised input (the input itself without a norm) is kept in 8 bits, one scale for 128 consecutive points of a channel,
    with one bit for each of the ReLU's decisions: 1.16 bytes a value instead of 4.  norm.training (or `training`, if given) decides
    between the batch's statistics (running statistics updated, as BatchNorm1d does) and the running ones.  1..1024 channels."""
    x = _gpu(x, "x", (torch.float32,))
    if x.dim() != 3 or 0 in x.shape:
        raise ValueError(f"x must be (B,K,L) with at least one value, got {tuple(x.shape)}")
    w = weight.squeeze(2) if weight.dim() == 3 and weight.size(2) == 1 else weight
    if w.dim() != 2 or w.size(1) != x.size(1):
        raise ValueError(f"weight must be (N,{x.size(1)}) or (N,{x.size(1)},1), got {tuple(weight.shape)}")
    if bias is not None and bias.shape != (w.size(0),):
        raise ValueError(f"bias must be ({w.size(0)},), got {tuple(bias.shape)}")
    for t, name in ((w, "weight"), (bias, "bias")):
        if t is not None and not (t.device == x.device and t.dtype == torch.float32):
            raise ValueError(f"{name} must be a float32 tensor on the input's GPU")
    return _Act8Linear.apply(x.contiguous(), w.contiguous(), None if bias is None else bias.contiguous(), *_norm_args(norm, x, training))


class _Act8NormRelu(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gamma, beta, running_mean, running_var, batches, momentum, eps):
        L_ = _lib.lib()
        B, C, L = x.shape
        dev = x.device
        nkept, nws = _act8_bytes("act8_norm_relu", B, C, L, True, 0)
        kept, ws = _bytes(nkept, dev), _bytes(nws, dev)
        y = torch.empty((B, C, L), dtype=torch.float32, device=dev)
        _call(L_.p2n_act8_norm_relu_forward, "p2n_act8_norm_relu_forward", dev, x.data_ptr(), B, C, L, gamma.data_ptr(), beta.data_ptr(),
              _rt.ptr(running_mean), _rt.ptr(running_var), _rt.ptr(batches), momentum, eps, y.data_ptr(), kept.data_ptr(), nkept,
              ws.data_ptr(), nws)
        _changed(running_mean, running_var, batches, momentum)
        ctx.save_for_backward(kept, gamma)
        ctx.meta = (B, C, L, momentum < 0)
        return y

    @staticmethod
    def backward(ctx, g):
        return _once(_Act8NormRelu, ctx, g) if torch.is_grad_enabled() else _Act8NormRelu.gradients(ctx, g)

    @staticmethod
    def gradients(ctx, g):
        kept, gamma = ctx.saved_tensors
        B, C, L, frozen = ctx.meta
        L_ = _lib.lib()
        g = g.contiguous()
        dev = g.device
        dx = torch.empty((B, C, L), dtype=torch.float32, device=dev)
        dgamma, dbeta = (torch.empty_like(gamma) if ctx.needs_input_grad[i] else None for i in (1, 2))
        nkept, nws = _act8_bytes("act8_norm_relu", B, C, L, True, 0)
        ws = _bytes(nws, dev)
        _call(L_.p2n_act8_norm_relu_backward, "p2n_act8_norm_relu_backward", dev, g.data_ptr(), B, C, L, gamma.data_ptr(), int(frozen),
              kept.data_ptr(), nkept, dx.data_ptr(), _rt.ptr(dgamma), _rt.ptr(dbeta), ws.data_ptr(), nws)
        return dx, dgamma, dbeta, None, None, None, None, None


def act8_norm_relu(x: torch.Tensor, norm: nn.BatchNorm1d, training: Optional[bool] = None) -> torch.Tensor:
    """x (B, C, L) float32 -> relu(norm(x)), differentiable in x and the norm's parameters; what the backward pass needs of x is
    kept in 8 bits and the ReLU's decisions as bits, as in act8_linear.  `training`, if given, in place of norm.training."""
    x = _gpu(x, "x", (torch.float32,))
    if x.dim() != 3 or 0 in x.shape:
        raise ValueError(f"x must be (B,C,L) with at least one value, got {tuple(x.shape)}")
    if norm is None:
        raise TypeError("norm must be a BatchNorm1d, got None")
    return _Act8NormRelu.apply(x.contiguous(), *_norm_args(norm, x, training))
