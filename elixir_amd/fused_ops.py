"""Layer norm and embedding of a training or serving step on the HIP kernels of ``libelx_ops.so``: the functions
``layer_norm`` and ``embedding``, and the modules ``FusedLayerNorm`` and ``FusedEmbedding`` that a model can use in place of
torch's and that ``ElixirModule(fused_ops=True)`` puts in place of them.

The reference swaps ``F.layer_norm`` for a third party's fused kernel (elixir/kernels/layernorm.py:1-10) and leaves the
embedding to torch.  Both functions take device tensors in fp32, fp16 or bf16, compute in fp32 and round once, run on the
current stream of the tensors' device, allocate what they return (and, in backward, a workspace) through torch's allocator,
synchronise nothing, and can be captured into a graph.  A gradient that is itself to be differentiated
(``create_graph=True``) and gradients for many at once (``is_grads_batched=True``) are computed by torch's own operators; forward-mode derivatives and tracing are refused.  What the
functions cannot take they refuse; the modules fall back to torch instead, so that a model keeps running wherever it ran."""
from typing import Optional, Sequence, Union

import torch
import torch.nn as nn
from torch.autograd import forward_ad

from . import _ops_abi, _torch_ext

_DTYPES = (torch.float32, torch.float16, torch.bfloat16)
_MAX_TOKENS, _MAX_ROWS, _MAX_COLS, _MAX_ELEMS = 1 << 26, 1 << 30, 1 << 20, 1 << 34    # of an embedding
_ext = None


def _load():
    global _ext
    _ext = _torch_ext.load()
    return _ext


def layer_norm(input: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, eps: float = 1e-5,
               normalized_shape: Optional[Union[int, Sequence[int]]] = None) -> torch.Tensor:
    """Layer norm over the trailing dimensions ``normalized_shape`` (default: those of ``weight`` or ``bias``, else the last
    one): ``(x - mean) / sqrt(var + eps) * weight + bias`` with the variance of the whole row (no correction).

    input: device tensor in fp32, fp16 or bf16 with up to 16,384 elements per row; rows may lie apart (a slice of a
        wider tensor is read in place).  weight, bias: the same type and device, of shape ``normalized_shape``, or None.
    Returns a new contiguous tensor.  Differentiable in all three."""
    if isinstance(normalized_shape, int):
        normalized_shape = (normalized_shape, )
    return (_ext or _load()).layer_norm(input, weight, bias, eps, normalized_shape)


def embedding(input: torch.Tensor, weight: torch.Tensor, padding_idx: Optional[int] = None, scale: float = 1.0) -> torch.Tensor:
    """Rows of ``weight`` named by ``input``, times ``scale`` (multiplied in fp32, rounded once).

    input: int64 or int32 device tensor of any shape, up to 2^26 tokens.  weight: [rows, cols] on the same device in fp32,
        fp16 or bf16; it and the embedded tokens have up to 2^34 elements.  padding_idx: a row whose tokens add nothing to
        the gradient (negative: counted from the end).
    The gradient of ``weight`` is dense, summed in fp32 in a fixed order (the same bits every time) and rounded
    once.  The indices are not checked on the host: one outside the table gives a row of NaN and no gradient."""
    return (_ext or _load()).embedding(input, weight, padding_idx, scale)


# --------------------------------------------------------------------------------------------------------------- modules


def _plain_eager(*tensors: Optional[torch.Tensor]) -> bool:
    """Ordinary device tensors of a supported type, outside of autocast, of tracing and other dispatch modes, of functorch
    transforms and of forward-mode derivatives: everything else is torch's."""
    if (torch.compiler.is_compiling() or torch.is_autocast_enabled() or torch._C._are_functorch_transforms_active()
            or torch.jit.is_tracing() or torch._C._len_torch_dispatch_stack() or forward_ad._current_level >= 0):
        return False
    for t in tensors:
        if t is not None and not (type(t) in (torch.Tensor, nn.Parameter) and t.is_cuda and t.layout == torch.strided):
            return False
    return True


class FusedLayerNorm(nn.LayerNorm):
    """``nn.LayerNorm`` on ``layer_norm``.  Same parameters, same state; inputs that function does not take (other types or
    devices, more than 16,384 elements per row, autocast, compiled, traced or transformed code, forward-mode derivatives) go
    to torch."""

    def forward(self, input: torch.Tensor) -> torch.Tensor:
        w, b = self.weight, self.bias
        cols = 1
        for s in self.normalized_shape:
            cols *= s
        if (_plain_eager(input, w, b) and input.dtype in _DTYPES and all(t is None or t.dtype == input.dtype and t.device == input.device
                                                                        for t in (w, b))
                and 1 <= cols <= _ops_abi.layer_norm_max_cols()
                and tuple(input.shape[-len(self.normalized_shape):]) == tuple(self.normalized_shape)):
            return layer_norm(input, w, b, self.eps, self.normalized_shape)
        return super().forward(input)


class FusedEmbedding(nn.Embedding):
    """``nn.Embedding`` on ``embedding``, with a factor on the embedded rows (``scale``).  Same parameters, same state;
    ``max_norm``, ``scale_grad_by_freq`` and ``sparse``, other types or devices, autocast, compiled, traced or transformed
    code and forward-mode derivatives go to torch (and are scaled after it)."""

    scale: float = 1.0    # also that of a module which was an nn.Embedding before

    def __init__(self, *args, scale: float = 1.0, **kwargs):
        super().__init__(*args, **kwargs)
        self.scale = float(scale)

    def forward(self, input: torch.Tensor) -> torch.Tensor:
        w = self.weight
        if (_plain_eager(input, w) and self.max_norm is None and not self.scale_grad_by_freq and not self.sparse and w.dtype in _DTYPES
                and input.dtype in (torch.int64, torch.int32) and w.device == input.device and input.numel() <= _MAX_TOKENS
                and 0 < w.shape[0] <= _MAX_ROWS and w.shape[1] <= _MAX_COLS and w.numel() <= _MAX_ELEMS
                and input.numel() * w.shape[1] <= _MAX_ELEMS):
            return embedding(input, w, self.padding_idx, self.scale)
        out = super().forward(input)
        return out if self.scale == 1.0 else out * self.scale


_SWAPS = {nn.LayerNorm: FusedLayerNorm, nn.Embedding: FusedEmbedding}


def fuse_modules(module: nn.Module) -> int:
    """Turns every ``nn.LayerNorm`` and ``nn.Embedding`` of ``module`` (exactly these classes, not subclasses) into the fused
    one, in place: the module objects, their parameters, hooks and state stay what they are.  Returns how many it turned."""
    count = 0
    for m in module.modules():
        fused = _SWAPS.get(type(m))
        if fused is not None and 'forward' not in m.__dict__:    # a forward of its own: somebody else's module by now
            m.__class__ = fused
            count += 1
    return count
