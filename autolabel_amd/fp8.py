"""Linear layers in 8-bit floating point with one power-of-two scale per block of 128 (csrc/fp8.hip), and their gradients.

The wide feature heads (autolabel/models.py:117-136 at LSeg width) and the compression autoencoder (autolabel/models.py:268-294) are matrix
products over up to a million rows; the reference runs them in fp16.  Here an operand is cut into blocks of 128 along the contracted axis and
each block is held as 8-bit values (``'e4m3'``, or ``'e5m2'`` with more range and a bit less precision) times one power of two, chosen so that
nothing is clipped; the products run on the block-scaled matrix instructions and accumulate in fp32.

    w = fp8.quantize(weight)                 # [out, in], once
    y = fp8.linear(x, w, relu=True)          # x [..., in] fp16 / bf16 / fp32 -> [..., out]
    dx, dw = fp8.linear_backward(g, x, fp8.quantize(weight, transpose=True))

``Linear`` wraps the three for autograd.  Every call allocates its results and its scratch from torch's allocator and enqueues on the current
stream of the tensors' device; nothing is kept between calls and nothing synchronises, so the calls can be captured into a graph.
"""
import contextlib
import functools
from dataclasses import dataclass

import torch

from . import hip as H

BLOCK = 128
FORMATS = {'e4m3': (0, torch.float8_e4m3fn), 'e5m2': (1, torch.float8_e5m2)}
TYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
MOST = (1 << 31) - 256       # rows and columns (the C entry points count them, and tiles of them, in 32 bits)


def _blocks(n):
    return (n + BLOCK - 1) // BLOCK


@dataclass
class Fp8Blocks:
    """A matrix [rows, cols] in 8-bit blocks: ``q`` [rows, >= 128 ceil(cols / 128)] of the 8-bit type (zeros behind column ``cols``) and
    ``scale`` [rows, a multiple of 4 >= ceil(cols / 128)] uint8, exponent + 127 of each block's power of two."""
    q: torch.Tensor
    scale: torch.Tensor
    cols: int
    fmt: str = 'e4m3'

    @property
    def rows(self):
        return self.q.shape[0]

    def dequantize(self):
        """The values the blocks stand for, [rows, cols] fp32 (torch operations: for inspection)."""
        s = ((self.scale.int()) << 23).view(torch.float32)[:, :_blocks(self.cols)]
        return (self.q.float()[:, :_blocks(self.cols) * BLOCK].reshape(self.rows, -1, BLOCK) * s[..., None]).reshape(self.rows, -1)[:, :self.cols]

    def _check(self, name):
        if self.fmt not in FORMATS:
            raise ValueError(f'{name}: unknown 8-bit format {self.fmt!r} (one of {", ".join(FORMATS)})')
        nb = _blocks(self.cols)
        q, s = self.q, self.scale
        shape = q.shape
        if self.cols < 1 or len(shape) != 2 or q.dtype is not FORMATS[self.fmt][1] or not q.is_contiguous() or shape[1] < nb * BLOCK or shape[1] % 16:
            raise ValueError(f'{name}: q must be contiguous {FORMATS[self.fmt][1]} [rows, whole blocks of 128 for {self.cols} columns], got {q.dtype} {tuple(q.shape)}')
        words = s.shape
        if len(words) != 2 or s.dtype is not torch.uint8 or not s.is_contiguous() or words[0] != shape[0] or words[1] < nb or words[1] % 4 or s.get_device() != q.get_device():
            raise ValueError(f'{name}: scale must be contiguous uint8 [rows, a multiple of 4 >= {nb}] beside q, got {s.dtype} {tuple(s.shape)}')
        if shape[0] > MOST or self.cols > MOST:
            raise ValueError(f'{name}: {shape[0]} rows of {self.cols} columns: neither may be more than {MOST}')


def _need(ok, message):
    if not ok:
        raise ValueError(message)


def _rows(name, x):
    """x as [rows, columns] with unit column stride (a view where its strides allow one, else a copy)."""
    if not isinstance(x, torch.Tensor) or x.dtype not in TYPES:
        raise ValueError(f'{name}: needs an fp16, bf16 or fp32 tensor')
    shape = x.shape
    if not shape or not shape[-1]:
        raise ValueError(f'{name}: needs at least one column, got shape {tuple(shape)}')
    if shape[-1] > MOST:
        raise ValueError(f'{name}: {shape[-1]} columns are more than {MOST}')
    if len(shape) != 2:
        x = x.detach().reshape(-1, shape[-1])
    if x.stride(1) != 1 and shape[-1] > 1:
        x = x.detach().contiguous()
    return x


def _pitch(x):
    return x.stride(0) if x.shape[0] > 1 else x.shape[1]


_NOTHING = contextlib.nullcontext()


def _on(a, b=None):
    """The tensors' common device made current (a no-op where it is)."""
    i = a.get_device()
    if i < 0 or (b is not None and b.get_device() != i):
        if i < 0 or b.get_device() < 0:
            raise ValueError('autolabel_amd.fp8 has no CPU path: needs device tensors')
        raise ValueError(f'tensors on different devices: {a.device} and {b.device}')
    return _NOTHING if i == torch.cuda.current_device() else torch.cuda.device(i)


# (functions of the sizes alone)
@functools.lru_cache(maxsize=4096)
def _linear_ws_bytes(*sizes):
    return H.lib().aln_fp8_linear_ws_bytes(*sizes)


@functools.lru_cache(maxsize=4096)
def _grad_weight_ws_bytes(*sizes):
    return H.lib().aln_fp8_grad_weight_ws_bytes(*sizes)


def _p(t):
    return t.data_ptr()


def _empty_blocks(rows, cols, fmt, device):
    nb = _blocks(cols)
    return Fp8Blocks(torch.empty(rows, nb * BLOCK, dtype=FORMATS[fmt][1], device=device),
                     torch.empty(rows, (nb + 3) // 4 * 4, dtype=torch.uint8, device=device), cols, fmt)


def quantize(x, fmt='e4m3', transpose=False):
    """Blocks of ``x`` [..., K] along its last axis -> Fp8Blocks of [rows, K]; ``transpose=True``: blocks of x^T along the rows of x ->
    Fp8Blocks of [K, rows] (what a product over the rows needs).  Blocks carry no gradient."""
    _need(fmt in FORMATS, f'quantize: unknown 8-bit format {fmt!r} (one of {", ".join(FORMATS)})')
    x = _rows('quantize', x)
    m, k = x.shape
    _need(m >= 1 or not transpose, 'quantize: x^T of an empty x has no columns')
    with _on(x):
        out = _empty_blocks(k, m, fmt, x.device) if transpose else _empty_blocks(m, k, fmt, x.device)
        H.call('aln_fp8_quantize_t' if transpose else 'aln_fp8_quantize', _p(x), TYPES[x.dtype], _pitch(x), m, k, FORMATS[fmt][0], _p(out.q),
               out.q.shape[1], _p(out.scale), out.scale.shape[1], H.raw_stream())
    return out


def _out_type(name, dtype):
    _need(dtype in TYPES, f'{name}: results are fp16, bf16 or fp32, not {dtype}')
    return dtype


def matmul(a, b, out_dtype=torch.float16, relu=False):
    """a [M, K] b [N, K]^T of two Fp8Blocks -> [M, N], accumulated in fp32 and rounded once."""
    a._check('matmul: a'); b._check('matmul: b')
    _need(a.cols == b.cols, f'matmul: the operands contract over {a.cols} and {b.cols} columns')
    _need(b.rows >= 1, 'matmul: b has no rows')
    _out_type('matmul', out_dtype)
    m, n, k = a.rows, b.rows, a.cols
    with _on(a.q, b.q):
        y = torch.empty(m, n, dtype=out_dtype, device=a.q.device)
        nbytes = int(H.lib().aln_fp8_nt_ws_bytes(m, n, k))
        ws = torch.empty(nbytes, dtype=torch.uint8, device=a.q.device) if nbytes else None
        H.call('aln_fp8_nt', _p(a.q), a.q.shape[1], _p(a.scale), a.scale.shape[1], FORMATS[a.fmt][0], _p(b.q), b.q.shape[1], _p(b.scale),
               b.scale.shape[1], FORMATS[b.fmt][0], m, n, k, _p(y), n, TYPES[out_dtype], int(bool(relu)), _p(ws) if nbytes else None, nbytes, H.raw_stream())
    return y


def linear(x, weight, relu=False, out_dtype=None, fmt='e4m3', out=None):
    """x [..., K] W^T for ``weight`` = Fp8Blocks of W [N, K] -> [..., N] of x's type (or ``out_dtype``); the rows of x are cut into blocks of
    ``fmt`` on the way.  (In a 16-bit result each term may be off by 2^-13 of the
    largest of its 64; in an fp32 result, at about half the rate, the terms are exact.)  ``relu``: negative results become 0.  ``out``: a contiguous tensor of the result's shape to write it into (its type
    decides the result's); it must not overlap x.  The result carries no gradient: while gradients are tracked, an x that requires one is refused
    (``Linear`` is the layer with its gradients)."""
    if isinstance(x, torch.Tensor) and x.requires_grad and torch.is_grad_enabled():
        raise ValueError('linear: x requires a gradient, which the result would not carry: use fp8.Linear, x.detach(), or call under torch.no_grad()')
    return _linear(x, weight, relu, out_dtype, fmt, out)


def _linear(x, weight, relu=False, out_dtype=None, fmt='e4m3', out=None):
    if not isinstance(weight, Fp8Blocks):
        raise ValueError('linear: weight must be Fp8Blocks (fp8.quantize)')
    weight._check('linear: weight')
    if fmt not in FORMATS:
        raise ValueError(f'linear: unknown 8-bit format {fmt!r} (one of {", ".join(FORMATS)})')
    rows = _rows('linear', x)
    (m, k), (n, ldw) = rows.shape, weight.q.shape
    if k != weight.cols or n < 1:
        raise ValueError(f'linear: x has {k} columns, the weight {n} rows of {weight.cols} columns')
    if out is not None:
        if not torch.is_tensor(out) or out.shape != (*x.shape[:-1], n) or not out.is_contiguous() or out.get_device() != x.get_device() or out_dtype not in (None, out.dtype):
            raise ValueError(f'linear: out must be a contiguous tensor of shape {(*x.shape[:-1], n)} beside x (of out_dtype, where given)')
        if out.requires_grad and torch.is_grad_enabled():
            raise ValueError('linear: out must not require a gradient (autograd does not see what is written into it)')
        out_dtype = out.dtype
    if out_dtype is None:
        out_dtype = x.dtype
    elif out_dtype not in TYPES:
        raise ValueError(f'linear: results are fp16, bf16 or fp32, not {out_dtype}')
    if rows.stride(0) >= 1 << 25:      # (rows very far apart)
        rows = rows.detach().clone(memory_format=torch.contiguous_format)
    if out is not None and m and rows.data_ptr() < out.data_ptr() + out.nbytes and out.data_ptr() < rows.data_ptr() + ((m - 1) * rows.stride(0) + k) * rows.element_size():
        raise ValueError('linear: out must not overlap x')
    with _on(rows, weight.q):
        y = torch.empty(*x.shape[:-1], n, dtype=out_dtype, device=x.device) if out is None else out
        x_type, y_type, fmt_w = TYPES[x.dtype], TYPES[out_dtype], FORMATS[weight.fmt][0]
        nbytes = _linear_ws_bytes(m, n, k, x_type, y_type, fmt_w)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device) if nbytes else None
        H.call('aln_fp8_linear', rows.data_ptr(), x_type, _pitch(rows), FORMATS[fmt][0], weight.q.data_ptr(), ldw, weight.scale.data_ptr(),
               weight.scale.shape[1], fmt_w, m, n, k, y.data_ptr(), n, y_type, 1 if relu else 0, ws.data_ptr() if nbytes else None, nbytes, H.raw_stream())
    if out is not None and not out.is_inference():
        torch.autograd.graph.increment_version(out)      # (a backward pass that saved it notices)
    return y


def linear_backward(g, x, weight_t, grad_fmt='e4m3', need_dx=True, need_dw=True):
    """Gradients of y = x W^T (no activation) from ``g`` = dL/dy [..., N] and ``x`` [..., K]: (dL/dx of x's type, dL/dW [N, K] fp32), either
    one None where not needed.  ``weight_t`` = Fp8Blocks of W^T [K, N] (not read for dL/dW alone: may be None then).  g is cut into blocks of
    ``grad_fmt`` along N for dL/dx, g and x along their rows for dL/dW; the sums over the rows are taken in a fixed order.  The gradients are not
    tracked themselves (no second derivatives)."""
    if grad_fmt not in FORMATS:
        raise ValueError(f'linear_backward: unknown 8-bit format {grad_fmt!r} (one of {", ".join(FORMATS)})')
    gr, xr = _rows('linear_backward: g', g), _rows('linear_backward: x', x)
    if g.shape[:-1] != x.shape[:-1]:
        raise ValueError(f'linear_backward: g has the rows {tuple(g.shape[:-1])}, x {tuple(x.shape[:-1])}')
    (m, n), k = gr.shape, xr.shape[1]
    dx = dw = None
    if need_dx:
        if not isinstance(weight_t, Fp8Blocks):
            raise ValueError('linear_backward: weight_t must be Fp8Blocks (fp8.quantize of the transposed weight)')
        weight_t._check('linear_backward: weight_t')
        if weight_t.rows != k or weight_t.cols != n:
            raise ValueError(f'linear_backward: weight_t is {weight_t.rows} x {weight_t.cols}, x has {k} columns and g {n}')
        dx = _linear(gr, weight_t, out_dtype=x.dtype, fmt=grad_fmt)
        if len(x.shape) != 2:
            dx = dx.reshape(x.shape)
    if need_dw:
        if m > 1:       # (rows that overlap, as an expanded gradient's do, or lie very far apart)
            if not n <= gr.stride(0) < 1 << 24:
                gr = gr.detach().clone(memory_format=torch.contiguous_format)
            if not k <= xr.stride(0) < 1 << 24:
                xr = xr.detach().clone(memory_format=torch.contiguous_format)
        with _on(gr, xr):
            if m == 0:
                return dx, torch.zeros(n, k, dtype=torch.float32, device=x.device)
            dw = torch.empty(n, k, dtype=torch.float32, device=x.device)
            g_type, x_type = TYPES[g.dtype], TYPES[x.dtype]
            nbytes = _grad_weight_ws_bytes(m, n, k, g_type, x_type)
            ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device) if nbytes else None
            H.call('aln_fp8_grad_weight', gr.data_ptr(), g_type, _pitch(gr), FORMATS[grad_fmt][0], xr.data_ptr(), x_type, _pitch(xr), m, n, k,
                   dw.data_ptr(), ws.data_ptr() if nbytes else None, nbytes, H.raw_stream())
    return dx, dw


class _LinearFunction(torch.autograd.Function):

    @staticmethod
    def forward(ctx, x, weight, grad_fmt):
        ctx.save_for_backward(x, weight)
        ctx.grad_fmt = grad_fmt
        return linear(x, quantize(weight))

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        x, weight = ctx.saved_tensors
        need_dx, need_dw = ctx.needs_input_grad[:2]
        dx, dw = linear_backward(g, x, quantize(weight, transpose=True) if need_dx else None, ctx.grad_fmt, need_dx, need_dw)
        return dx, None if dw is None else dw.to(weight.dtype), None


class Linear(torch.nn.Linear):
    """``torch.nn.Linear`` without a bias whose three products run in 8-bit blocks: the same parameter, initialisation and state_dict, the
    weight kept in its own type and cut into blocks at every call (it changes with every optimizer step)."""

    def __init__(self, in_features, out_features, grad_fmt='e4m3', device=None, dtype=None):
        _need(grad_fmt in FORMATS, f'Linear: unknown 8-bit format {grad_fmt!r} (one of {", ".join(FORMATS)})')
        super().__init__(in_features, out_features, bias=False, device=device, dtype=dtype)
        self.grad_fmt = grad_fmt

    def forward(self, x):
        return _LinearFunction.apply(x, self.weight, self.grad_fmt)
