"""Linear layers in 8-bit integers on MI355X, for serving the dense network (`hubconf.MPMAE(..., int8=True)`): weights quantised once per output
channel, activations per row (token, pixel) inside the call, exact integer sums on the matrix cores, scales and bias applied on the way out.

    w = quantize_weight(layer.weight, layer.bias)      # once
    y = linear_int8(x, w)                              # [..., K] fp32 / bf16 / fp16 -> [..., N] of the same type
    quantize_model(model)                              # every nn.Linear of a module tree, in place

    x_q = round(127 x / max|x|), s_x = max|x| / 127 per row;  y = s_x s_w (x_q w_q^T) + bias

Inference only: an input that requires a gradient or carries a tangent is refused. The call is an operator of torch's dispatcher, so traces and exported graphs
hold it; `load_ops()` before loading one. There is no CPU form.
"""
import torch
import torch.nn as nn

from . import _lib

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
MAX_K = 131071          # 127 * 127 * K fits 32 bits


def _rows(x, k):
    """x as rows of k elements that lie next to each other: (tensor that owns them, rows, elements from row to row)."""
    if x.dim() != 2 or (x.stride(1) != 1 and k > 1):
        x = x.reshape(-1, k)
        if x.stride(1) != 1 and k > 1:
            x = x.contiguous()
    return x, x.shape[0], x.stride(0)


_linear = None          # native call, from the first use on


def load_ops():
    """Registers the operators that a traced or exported network calls (`torch.ops.mpmae.linear_int8`): before `torch.jit.load` of one. `linear_int8` does it by
    itself."""
    global _linear
    _linear = _lib.host_tensors().linear_i8
    return _linear


class Int8Weight:
    """A weight matrix [N, K] as int8 codes with one scale per row, laid out for `linear_int8`. Made by `quantize_weight`."""

    def __init__(self, q, scale, bias, k):
        self.q, self.scale, self.bias, self.k, self.n = q, scale, bias, k, q.shape[0]
        self.device = q.device

    def dequantize(self):
        """The fp32 matrix that the codes stand for."""
        return self.q[:, :self.k].float() * self.scale[:, None]


@torch.no_grad()
def quantize_weight(weight, bias=None):
    """weight [N, K] fp32 / bf16 / fp16 (and bias [N]) of a linear layer on the GPU -> Int8Weight."""
    if weight.dim() != 2 or 0 in weight.shape:
        raise ValueError(f"a weight is a matrix [N, K] with at least one element, not {tuple(weight.shape)}")
    if weight.dtype not in _DTYPES:
        raise ValueError(f"weights are fp32, bf16 or fp16, not {weight.dtype}")
    if weight.shape[1] > MAX_K:
        raise ValueError(f"rows of at most {MAX_K} elements: their integer sums fit 32 bits")
    if bias is not None and (bias.shape != weight.shape[:1] or bias.dtype not in _DTYPES or bias.device != weight.device):
        raise ValueError(f"a bias is a floating vector [{weight.shape[0]}] on the weight's device")
    if weight.device.type != "cuda":
        raise ValueError(f"this layer runs on the GPU only: the weight is on {weight.device}")
    load_ops()
    k = int(weight.shape[1])
    q, scale = torch.ops.mpmae.quantize_int8(_rows(weight.detach(), k)[0])
    # (a copy of the bias too: the codes are those of this moment)
    return Int8Weight(q, scale, None if bias is None else bias.detach().to(torch.float32, copy=True).contiguous(), k)


def linear_int8(x, w):
    """y = x W^T + bias for x [..., K] fp32 / bf16 / fp16 on the weight's GPU; y has x's type. A row that holds NaN or infinity gives a row of NaN."""
    return (_linear or load_ops())(x, w.q, w.scale, w.bias, w.k)          # torch.ops.mpmae.linear_int8 with less on the way: csrc/host_tensors.cpp


class Int8Linear(nn.Module):
    """nn.Linear with int8 weights, inference only. Codes, scales and bias are buffers: they are saved, loaded and moved with the model; `.half()` and
    the like leave them in their own types."""

    def __init__(self, in_features, out_features, bias=True, device=None):
        super().__init__()
        self.in_features, self.out_features, self._weight = in_features, out_features, None
        kp = -(-in_features // _lib.I8_KPAD) * _lib.I8_KPAD
        self.register_buffer("q", torch.zeros(out_features, kp, dtype=torch.int8, device=device))
        self.register_buffer("scale", torch.zeros(out_features, dtype=torch.float32, device=device))
        self.register_buffer("bias", torch.zeros(out_features, dtype=torch.float32, device=device) if bias else None)

    @classmethod
    def from_linear(cls, linear):
        w = quantize_weight(linear.weight, linear.bias)
        self = cls(linear.in_features, linear.out_features, linear.bias is not None, device="meta")
        self.q, self.scale, self.bias = w.q, w.scale, w.bias
        self.training = linear.training
        for name in _FORWARD_HOOKS:          # (the dictionaries themselves: handles of `register_forward_hook` go on removing from them)
            setattr(self, name, getattr(linear, name))
        return self

    def _apply(self, fn, recurse=True):
        for name, buf in self._buffers.items():
            if buf is not None:
                moved = fn(buf)
                self._buffers[name] = moved if moved.dtype == buf.dtype else buf.to(moved.device)
        return self

    def forward(self, x):
        w = self._weight
        if w is None or w.q is not self.q or w.scale is not self.scale or w.bias is not self.bias:
            w = self._weight = Int8Weight(self.q, self.scale, self.bias, self.in_features)
        return linear_int8(x, w)

    def extra_repr(self):
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}"


_FORWARD_HOOKS = ("_forward_hooks", "_forward_hooks_with_kwargs", "_forward_hooks_always_called", "_forward_pre_hooks", "_forward_pre_hooks_with_kwargs")


def _plain(module):
    """Whether a module is an nn.Linear and nothing more: no subclass (its users may read the weight), no weight that a hook computes (weight norm, pruning), no
    forward of its own."""
    return type(module) is nn.Linear and module._parameters.get("weight") is not None and "forward" not in module.__dict__


def quantize_model(model):
    """Every plain nn.Linear of the module tree (on the GPU) becomes an Int8Linear, in place, and takes its forward hooks along; one that is used in several
    places stays one, others stay as they are. Returns the model. Nothing is replaced unless every layer can be."""
    made = {m: Int8Linear.from_linear(m) for m in model.modules() if _plain(m)}
    for parent in list(model.modules()):
        for name, child in parent._modules.items():
            if child in made:
                parent._modules[name] = made[child]
    return made.get(model, model)
