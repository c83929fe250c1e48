"""Layer norm and embedding of a training or serving step on the HIP kernels of ``libelx_ops.so``: the functions
``layer_norm`` and ``embedding``, and the modules ``FusedLayerNorm`` and ``FusedEmbedding`` that a model can use in place of
torch's and that ``ElixirModule(fused_ops=True)`` puts in place of them.

The reference swaps ``F.layer_norm`` for a third party's fused kernel (elixir/kernels/layernorm.py:1-10) and leaves the
embedding to torch.  Both functions take device tensors in fp32, fp16 or bf16, compute in fp32 and round once, run on the
current stream of the tensors' device, allocate what they return (and, in backward, a workspace) through torch's allocator,
synchronise nothing, and can be captured into a graph.  A gradient that is itself to be differentiated
(``create_graph=True``) is computed by torch's own operators.  What the functions cannot take they refuse; the modules fall
back to torch instead, so that a model keeps running wherever it ran."""
from typing import Optional, Sequence, Tuple, Union

import torch
import torch.nn as nn
import torch.nn.functional as F

from . import _abi, _ops_abi

_CODES = {torch.float32: _abi.ELX_F32, torch.float16: _abi.ELX_F16, torch.bfloat16: _abi.ELX_BF16}


def _rows(x: torch.Tensor, cols: int) -> Tuple[torch.Tensor, int]:
    """``x`` as rows of ``cols`` elements: the tensor to read them from and the distance of two rows.  A tensor whose rows
    do not lie at one distance, or whose elements do not lie side by side, is copied."""
    if x.is_contiguous():
        return x, cols
    if x.dim() >= 2 and x.stride(-1) == 1 or x.shape[-1] == 1:
        step, ok = None, x.shape[-1] == cols
        expect = None
        for size, stride in zip(reversed(x.shape[:-1]), reversed(x.stride()[:-1])):    # from the innermost row dimension out
            if size == 1:
                continue
            if expect is None:
                step, expect = stride, stride * size
            elif stride != expect:
                ok = False
                break
            else:
                expect = stride * size
        if ok and (step is None or step >= cols):
            return x, cols if step is None else step
    return x.contiguous(), cols


def _check_device(name: str, *tensors: Optional[torch.Tensor]) -> torch.device:
    device = tensors[0].device
    for t in tensors:
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError(f'{name} runs on the GPU: its tensors must live in device memory')
        if t.device != device:
            raise RuntimeError(f'{name}: tensors on {device} and {t.device}')
    return device


def _check_dtype(name: str, *tensors: Optional[torch.Tensor]) -> int:
    dtype = tensors[0].dtype
    if dtype not in _CODES:
        raise TypeError(f'{name} takes float32, float16 or bfloat16, not {dtype}')
    for t in tensors:
        if t is not None and t.dtype != dtype:
            raise TypeError(f'{name}: tensors of {dtype} and {t.dtype}')
    return _CODES[dtype]


# ------------------------------------------------------------------------------------------------------------ layer norm


def _layer_norm_forward(x, weight, bias, cols, eps, keep):
    """(y, mean, rstd); the last two only with ``keep``."""
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    rows = x.numel() // cols
    mean = rstd = None
    if keep:
        mean, rstd = torch.empty(2, rows, dtype=torch.float32, device=x.device).unbind(0)
    if rows:
        src, stride = _rows(x, cols)
        weight = weight.contiguous() if weight is not None else None
        bias = bias.contiguous() if bias is not None else None
        with torch.cuda.device(x.device):
            _ops_abi.layer_norm_fwd(src.data_ptr(), weight.data_ptr() if weight is not None else 0,
                                    bias.data_ptr() if bias is not None else 0, y.data_ptr(), mean.data_ptr() if keep else 0,
                                    rstd.data_ptr() if keep else 0, rows, cols, stride, eps, _CODES[x.dtype],
                                    torch.cuda.current_stream(x.device).cuda_stream)
    return y, mean, rstd


class _LayerNorm(torch.autograd.Function):

    @staticmethod
    def forward(ctx, x, weight, bias, normalized, cols, eps):
        y, mean, rstd = _layer_norm_forward(x, weight, bias, cols, eps, True)
        ctx.save_for_backward(x, weight, mean, rstd)
        ctx.normalized, ctx.cols, ctx.eps = normalized, cols, eps
        return y

    @staticmethod
    def backward(ctx, dy):
        x, w, mean, rstd = ctx.saved_tensors
        cols = ctx.cols
        rows = x.numel() // cols
        want_x, want_w, want_b = ctx.needs_input_grad[:3]
        if torch.is_grad_enabled():    # the gradient is to be differentiated
            b = torch.zeros(ctx.normalized, dtype=x.dtype, device=x.device, requires_grad=True) if want_b else None
            leaves = [t for t, want in ((x, want_x), (w, want_w), (b, want_b)) if want]
            y = F.layer_norm(x, ctx.normalized, w, b, ctx.eps)
            grads = iter(torch.autograd.grad(y, leaves, dy, create_graph=True))
            return tuple(next(grads) if want else None for want in (want_x, want_w, want_b)) + (None, None, None)
        w = w.contiguous() if w is not None else None
        new = lambda shape: torch.empty(shape, dtype=x.dtype, device=x.device)    # noqa: E731
        dx = new(x.shape) if want_x else None
        dw = new(ctx.normalized) if want_w else None
        db = new(ctx.normalized) if want_b else None
        if rows == 0:
            return dx, dw.zero_() if want_w else None, db.zero_() if want_b else None, None, None, None
        if dx is None and dw is None and db is None:
            return None, None, None, None, None, None
        src, x_stride = _rows(x, cols)
        grad, dy_stride = _rows(dy, cols)
        nbytes = _ops_abi.layer_norm_bwd_workspace(rows, cols) if want_w or want_b else 0
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=x.device) if nbytes else None
        ptr = lambda t: t.data_ptr() if t is not None else 0    # noqa: E731
        with torch.cuda.device(x.device):
            _ops_abi.layer_norm_bwd(grad.data_ptr(), src.data_ptr(), ptr(w), mean.data_ptr(), rstd.data_ptr(), ptr(dx), ptr(dw), ptr(db),
                                    ptr(workspace), nbytes, rows, cols, dy_stride, x_stride, _CODES[x.dtype],
                                    torch.cuda.current_stream(x.device).cuda_stream)
        return dx, dw, db, None, None, None


def layer_norm(input: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, eps: float = 1e-5,
               normalized_shape: Optional[Union[int, Sequence[int]]] = None) -> torch.Tensor:
    """Layer norm over the trailing dimensions ``normalized_shape`` (default: those of ``weight`` or ``bias``, else the last
    one): ``(x - mean) / sqrt(var + eps) * weight + bias`` with the variance of the whole row (no correction).

    input: device tensor in fp32, fp16 or bf16 with up to 16,384 elements per row; rows may lie apart (a slice of a
        wider tensor is read in place).  weight, bias: the same type and device, of shape ``normalized_shape``, or None.
    Returns a new contiguous tensor.  Differentiable in all three."""
    if normalized_shape is None:
        like = weight if weight is not None else bias
        normalized_shape = tuple(like.shape) if like is not None else tuple(input.shape[-1:])
    shape = (normalized_shape, ) if isinstance(normalized_shape, int) else tuple(normalized_shape)
    if not shape or tuple(input.shape[-len(shape):]) != shape:
        raise ValueError(f'layer_norm over {list(shape)} of an input of shape {list(input.shape)}')
    for name, t in (('weight', weight), ('bias', bias)):
        if t is not None and tuple(t.shape) != shape:
            raise ValueError(f'layer_norm: {name} has shape {list(t.shape)}, not {list(shape)}')
    _check_device('layer_norm', input, weight, bias)
    _check_dtype('layer_norm', input, weight, bias)
    cols = 1
    for s in shape:
        cols *= s
    if not 1 <= cols <= _ops_abi.layer_norm_max_cols():
        raise ValueError(f'layer_norm takes rows of 1 to {_ops_abi.layer_norm_max_cols()} elements, not {cols}')
    eps = float(eps)
    if torch.is_grad_enabled() and (input.requires_grad or weight is not None and weight.requires_grad
                                    or bias is not None and bias.requires_grad):
        return _LayerNorm.apply(input, weight, bias, shape, cols, eps)
    return _layer_norm_forward(input, weight, bias, cols, eps, False)[0]


# ------------------------------------------------------------------------------------------------------------- embedding


def _embedding_forward(index, table, scale):
    y = torch.empty(index.shape + table.shape[1:], dtype=table.dtype, device=table.device)
    if y.numel():
        with torch.cuda.device(table.device):
            _ops_abi.embedding_fwd(index.data_ptr(), index.element_size(), index.numel(), table.data_ptr(), table.shape[0],
                                   table.shape[1], scale, y.data_ptr(), _CODES[table.dtype],
                                   torch.cuda.current_stream(table.device).cuda_stream)
    return y


class _Embedding(torch.autograd.Function):

    @staticmethod
    def forward(ctx, index, table, padding, scale):
        ctx.save_for_backward(index)
        ctx.like, ctx.padding, ctx.scale = (table.shape, table.dtype, table.device), padding, scale
        return _embedding_forward(index, table.contiguous(), scale)

    @staticmethod
    def backward(ctx, dy):
        index, = ctx.saved_tensors
        shape, dtype, device = ctx.like
        if torch.is_grad_enabled():    # the gradient is to be differentiated
            inside = (index >= 0) & (index < shape[0])
            table = torch.zeros(shape, dtype=dtype, device=device, requires_grad=True)
            y = F.embedding(index.where(inside, 0), table, ctx.padding if ctx.padding >= 0 else None)
            dy = (dy * ctx.scale).where(inside.unsqueeze(-1), 0)
            return None, torch.autograd.grad(y, table, dy, create_graph=True)[0], None, None
        dtable = torch.empty(shape, dtype=dtype, device=device)
        n, (vocab, cols) = index.numel(), shape
        if n == 0 or dtable.numel() == 0:
            return None, dtable.zero_(), None, None
        grad, stride = _rows(dy, cols)
        nbytes = _ops_abi.embedding_bwd_workspace(n, vocab, cols)
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=device)
        with torch.cuda.device(device):
            _ops_abi.embedding_bwd(index.data_ptr(), index.element_size(), n, grad.data_ptr(), stride, dtable.data_ptr(), vocab, cols,
                                   ctx.scale, ctx.padding, workspace.data_ptr(), nbytes, _CODES[dtype],
                                   torch.cuda.current_stream(device).cuda_stream)
        return None, dtable, None, None


_MAX_TOKENS, _MAX_ROWS, _MAX_COLS = 1 << 26, 1 << 30, 1 << 20


def embedding(input: torch.Tensor, weight: torch.Tensor, padding_idx: Optional[int] = None, scale: float = 1.0) -> torch.Tensor:
    """Rows of ``weight`` named by ``input``, times ``scale`` (multiplied in fp32, rounded once).

    input: int64 or int32 device tensor of any shape, up to 2^26 tokens.  weight: [rows, cols] on the same device in fp32,
        fp16 or bf16.  padding_idx: a row whose tokens add nothing to the gradient (negative: counted from the end).
    The gradient of ``weight`` is dense, summed in fp32 in the order of the tokens (the same bits every time) and rounded
    once.  The indices are not checked on the host: one outside the table gives a row of NaN and no gradient."""
    if weight.dim() != 2:
        raise ValueError(f'embedding takes a table of two dimensions, not {weight.dim()}')
    if input.dtype not in (torch.int64, torch.int32):
        raise TypeError(f'embedding takes int64 or int32 indices, not {input.dtype}')
    _check_device('embedding', weight, input)
    _check_dtype('embedding', weight)
    rows, cols = weight.shape
    if input.numel() > _MAX_TOKENS or rows > _MAX_ROWS or cols > _MAX_COLS or (rows == 0 and input.numel() > 0):
        raise ValueError(f'embedding takes up to {_MAX_TOKENS} tokens and a table of 1 to {_MAX_ROWS} rows of up to {_MAX_COLS} elements')
    padding = -1
    if padding_idx is not None:
        if not -rows <= padding_idx < rows:
            raise ValueError(f'padding_idx {padding_idx} lies outside a table of {rows} rows')
        padding = padding_idx % rows
    index = input.contiguous()
    if torch.is_grad_enabled() and weight.requires_grad:
        return _Embedding.apply(index, weight, padding, float(scale))
    return _embedding_forward(index, weight.contiguous(), float(scale))


# --------------------------------------------------------------------------------------------------------------- modules


def _plain_eager(*tensors: Optional[torch.Tensor]) -> bool:
    """Ordinary device tensors of a supported type, outside of autocast, of tracing and of functorch transforms: everything
    else is torch's."""
    if torch.compiler.is_compiling() or torch.is_autocast_enabled() or torch._C._are_functorch_transforms_active():
        return False
    for t in tensors:
        if t is not None and not (type(t) in (torch.Tensor, nn.Parameter) and t.is_cuda and t.layout == torch.strided):
            return False
    return True


class FusedLayerNorm(nn.LayerNorm):
    """``nn.LayerNorm`` on ``layer_norm``.  Same parameters, same state; inputs that function does not take (other types or
    devices, more than 16,384 elements per row, autocast, compiled or transformed code) go to torch."""

    def forward(self, input: torch.Tensor) -> torch.Tensor:
        w, b = self.weight, self.bias
        cols = 1
        for s in self.normalized_shape:
            cols *= s
        if (_plain_eager(input, w, b) and input.dtype in _CODES and all(t is None or t.dtype == input.dtype and t.device == input.device
                                                                        for t in (w, b))
                and 1 <= cols <= _ops_abi.layer_norm_max_cols()
                and tuple(input.shape[-len(self.normalized_shape):]) == tuple(self.normalized_shape)):
            return layer_norm(input, w, b, self.eps, self.normalized_shape)
        return super().forward(input)


class FusedEmbedding(nn.Embedding):
    """``nn.Embedding`` on ``embedding``, with a factor on the embedded rows (``scale``).  Same parameters, same state;
    ``max_norm``, ``scale_grad_by_freq`` and ``sparse``, other types or devices, autocast, compiled or transformed code go to
    torch (and are scaled after it)."""

    scale: float = 1.0    # also that of a module which was an nn.Embedding before

    def __init__(self, *args, scale: float = 1.0, **kwargs):
        super().__init__(*args, **kwargs)
        self.scale = float(scale)

    def forward(self, input: torch.Tensor) -> torch.Tensor:
        w = self.weight
        if (_plain_eager(input, w) and self.max_norm is None and not self.scale_grad_by_freq and not self.sparse and w.dtype in _CODES
                and input.dtype in (torch.int64, torch.int32) and w.device == input.device and input.numel() <= _MAX_TOKENS
                and 0 < w.shape[0] <= _MAX_ROWS and w.shape[1] <= _MAX_COLS):
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
