"""MXFP4: microscaled 4-bit floating point linear layers and gated block (tcgen05 ``kind::mxf4``).

32 consecutive values along the axis that a product sums over share one power-of-two scale (E8M0);
each value is an E2M1 code: 17/32 byte per value.  The reference has no 4-bit path; this stands
beside its int8 one (``quantize_fp_to_int8``, ``BitLinear``; fireflykernels.py:96-124):

* ``quantize_fp_to_mxfp4`` / ``quantize_fp_to_mxfp4_dual``: the quantiser, along one axis or along
  both from one read; ``MXFP4Tensor.dequantize`` goes back.
* ``mxfp4_matmul``: the product of two quantised matrices.
* ``mxfp4_linear``: ``y = Q(x)·Q(W)ᵀ + b``.  With a floating-point ``W`` it is a training op: the
  gradient passes straight through the quantiser, and both backward products are MXFP4 products
  too, each operand quantised along the axis that product sums over
  (``dx = Q(dy)·Q(Wᵀ)ᵀ``, ``dW = Q(dyᵀ)·Q(xᵀ)ᵀ``).  With an ``MXFP4Tensor`` it serves: the weight
  is laid out once and streamed at 17/32 byte per value.
* ``mxfp4_swiglu``: ``down(silu(g)·u)``, ``[g | u] = gate_up(x)``, likewise.  Without gradients the
  activation and h's quantisation run in the gate/up product's epilogue (hidden size a multiple of
  128; otherwise in a quantiser pass over gu).  g, u, h and their gradients are rounded to bf16
  between the products, in training and serving alike, so both compute the same numbers.

Products accumulate in fp32 and return bf16.
"""
from __future__ import annotations

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from . import _capi


class MXFP4Tensor:
    """A matrix [rows, cols] held in MXFP4 with its blocks along the columns.

    ``codes``: uint8 [rows, 16·ceil(cols/32)], two codes to a byte, the earlier in the low nibble;
    ``scales``: the E8M0 bytes in the tensor core's chunk order (``scale_bytes()`` gives them per
    block); ``transposed``: the same matrix quantised along its rows, as [cols, rows], or ``None``
    (what the gradient of a product's other operand needs)."""

    __slots__ = ("codes", "scales", "shape", "transposed")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, shape: tuple[int, int],
                 transposed: "MXFP4Tensor | None" = None):
        rows, cols = int(shape[0]), int(shape[1])
        want = (rows + 127) // 128 * 2 * ((cols + 255) // 256) * 512
        if (cols < 1 or codes.dtype != torch.uint8 or tuple(codes.shape) != (rows, (cols + 31) // 32 * 16)
                or not codes.is_contiguous()):
            raise ValueError(f"MXFP4 codes of a {rows} x {cols} matrix: contiguous uint8 [rows, 16*ceil(cols/32)], "
                             f"got {codes.dtype} {tuple(codes.shape)}")
        if scales.dtype != torch.uint8 or scales.numel() != want or not scales.is_contiguous():
            raise ValueError(f"MXFP4 scales of a {rows} x {cols} matrix: {want} contiguous uint8, "
                             f"got {scales.dtype} {tuple(scales.shape)}")
        if codes.device != scales.device:
            raise RuntimeError(f"tensors on different devices: {codes.device} and {scales.device}")
        if transposed is not None and transposed.shape != (cols, rows):
            raise ValueError(f"transposed form of a {rows} x {cols} matrix has shape {transposed.shape}")
        self.codes, self.scales, self.shape, self.transposed = codes, scales, (rows, cols), transposed

    @classmethod
    def _made(cls, pair, rows: int, cols: int, transposed=None) -> "MXFP4Tensor":
        """From a kernel's own output."""
        q = cls.__new__(cls)
        q.codes, q.scales = pair
        q.shape, q.transposed = (rows, cols), transposed
        return q

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def _pair(self):
        return self.codes, self.scales

    def dequantize(self, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        """The values the codes stand for, as bfloat16 (exact), float32 (exact) or float16."""
        return _capi.mxfp4_dequant(self.codes, self.scales, *self.shape, dtype)

    def scale_bytes(self) -> torch.Tensor:
        """The E8M0 scale byte of every block, uint8 [rows, ceil(cols/32)]."""
        rows, cols = self.shape
        if rows == 0:
            return self.scales.new_empty((0, (cols + 31) // 32))
        s = self.scales.view((rows + 127) // 128, -1, 32, 4, 4)  # row tile, chunk, row % 32, row / 32, block % 4
        s = s.permute(0, 3, 2, 1, 4).reshape((rows + 127) // 128 * 128, -1)
        return s[:rows, :(cols + 31) // 32].contiguous()

    def __repr__(self) -> str:
        return f"MXFP4Tensor({self.shape[0]} x {self.shape[1]}, device={self.device})"


def _matrix(x: torch.Tensor, what: str) -> torch.Tensor:
    if not isinstance(x, torch.Tensor) or x.dim() != 2:
        raise ValueError(f"{what} must be a 2-D tensor, got {tuple(x.shape) if isinstance(x, torch.Tensor) else type(x)}")
    if x.requires_grad:
        x = x.detach()
    return x if x.dtype in (torch.float32, torch.bfloat16, torch.float16) else x.float()


def quantize_fp_to_mxfp4(x: torch.Tensor, transposed: bool = False) -> MXFP4Tensor:
    """``x`` [R, C] quantised with blocks of 32 along its rows.  ``transposed``: also keep the form with
    blocks along its columns (``.transposed``), which a backward pass through a weight held in this
    format needs."""
    x = _matrix(x, "x")
    rows, cols, _ = _capi.mxfp4_quant(x, rows=True, cols=transposed)
    R, C = x.shape
    return MXFP4Tensor._made(rows, R, C, MXFP4Tensor._made(cols, C, R) if transposed else None)


def quantize_fp_to_mxfp4_dual(x: torch.Tensor) -> tuple[MXFP4Tensor, MXFP4Tensor]:
    """``x`` [R, C] quantised along its rows and, as the matrix [C, R], along its columns: one read."""
    q = quantize_fp_to_mxfp4(x, transposed=True)
    qt, q.transposed = q.transposed, None
    return q, qt


def mxfp4_matmul(a: MXFP4Tensor, b: MXFP4Tensor, bias: torch.Tensor | None = None,
                 out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``a·bᵀ (+ bias)``: a [M, K], b [N, K] -> [M, N] in bfloat16 or float32."""
    if not isinstance(a, MXFP4Tensor) or not isinstance(b, MXFP4Tensor):
        raise ValueError("mxfp4_matmul takes two MXFP4Tensor operands")
    if a.shape[1] != b.shape[1]:
        raise ValueError(f"mxfp4_matmul: {a.shape} and {b.shape} differ in their contraction")
    return _product(a._pair(), b._pair(), a.shape[0], b.shape[0], a.shape[1], _bias(bias, b.shape[0]), out_dtype)


def _bias(bias: torch.Tensor | None, n: int) -> torch.Tensor | None:
    if bias is None:
        return None
    if tuple(bias.shape) != (n,):
        raise ValueError(f"bias must have shape ({n},), got {tuple(bias.shape)}")
    if bias.requires_grad:
        bias = bias.detach()
    return bias if bias.dtype == torch.float32 and bias.is_contiguous() else bias.to(torch.float32).contiguous()


def _product(a, b, M, N, K, bias=None, dtype=torch.bfloat16) -> torch.Tensor:
    """The product in ``dtype``: bf16 and fp32 from the kernel, fp16 rounded from its fp32 output."""
    if dtype in (torch.bfloat16, torch.float32):
        return _capi.mxfp4_gemm(a, b, M, N, K, bias, dtype)
    return _capi.mxfp4_gemm(a, b, M, N, K, bias, torch.float32).to(dtype)


def _weight_codes(w, need_t: bool, what: str):
    """Codes of a weight for the forward product and (``need_t``) for the product of its gradient."""
    if isinstance(w, MXFP4Tensor):
        if need_t and w.transposed is None:
            raise ValueError(f"the gradient through an MXFP4 {what} needs its transposed form: "
                             "quantize_fp_to_mxfp4(w, transposed=True)")
        return w._pair(), w.transposed._pair() if need_t else None
    rows, cols, _ = _capi.mxfp4_quant(_matrix(w, what), rows=True, cols=need_t)
    return rows, cols


class MXFP4LinearFn(torch.autograd.Function):
    """``Q(x)·Q(W)ᵀ + b`` and its straight-through gradient in MXFP4 products."""

    @staticmethod
    def forward(ctx, x, weight, bias, packed, grad):
        w = packed if packed is not None else weight
        O, K = w.shape
        T = x.shape[0]
        need_dx, need_dw = grad and ctx.needs_input_grad[0], grad and ctx.needs_input_grad[1]
        b = _bias(bias, O)
        ctx.dims, ctx.dtypes = (T, O, K), (x.dtype, None if packed is not None else weight.dtype,
                                           None if bias is None else bias.dtype)
        ctx.whole = packed is None and T > 0 and O > 0
        if ctx.whole:  # one call
            ctx.had = need_dx, need_dw
            y, saved = _capi.mxfp4_linear_train(_matrix(x, "x"), _matrix(weight, "weight"), b, need_dx, need_dw)
            ctx.save_for_backward(saved)
            return y
        if T == 0:
            ctx.save_for_backward(None, None, None, None)
            return torch.empty((0, O), dtype=torch.bfloat16, device=x.device)
        qx, qxt, _ = _capi.mxfp4_quant(_matrix(x, "x"), rows=True, cols=need_dw)
        qw, qwt = _weight_codes(w, need_dx, "weight")
        ctx.save_for_backward(*(qxt or (None, None)), *(qwt or (None, None)))
        return _product(qx, qw, T, O, K, b)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        T, O, K = ctx.dims
        xd, wd, bd = ctx.dtypes
        need_dx, need_dw, need_db = ctx.needs_input_grad[:3]
        dev = dy.device
        if T == 0 or O == 0:
            return (torch.zeros((T, K), dtype=xd, device=dev) if need_dx else None,
                    torch.zeros((O, K), dtype=wd, device=dev) if need_dw else None,
                    torch.zeros((O,), dtype=bd, device=dev) if need_db else None, None, None)
        if ctx.whole:
            dx, dw, db = _capi.mxfp4_linear_bwd(_matrix(dy, "dy"), ctx.saved_tensors[0], ctx.dims, *ctx.had,
                                                xd if need_dx else None, wd if need_dw else None, need_db)
            return dx, dw, db.to(bd) if need_db else None, None, None
        qxt, sxt, qwt, swt = ctx.saved_tensors
        q, qt, db = _capi.mxfp4_quant(_matrix(dy, "dy"), rows=need_dx, cols=need_dw, colsum=need_db)
        dx = _product(q, (qwt, swt), T, K, O, None, xd) if need_dx else None
        dw = _product(qt, (qxt, sxt), O, K, T, None, wd) if need_dw else None
        return dx, dw, db.to(bd) if need_db else None, None, None


class MXFP4SwiGLUFn(torch.autograd.Function):
    """The gated block ``down(silu(g)·u)``, ``[g | u] = gate_up(x)``, and its gradient."""

    @staticmethod
    def forward(ctx, x, gate_up, down, packed, grad):
        wgu, wd = (p if p is not None else w for p, w in zip(packed, (gate_up, down)))
        O, F = wd.shape
        T, K = x.shape
        need_dx, need_gu, need_d = (grad and n for n in ctx.needs_input_grad[:3])
        need = need_dx or need_gu or need_d
        need_dgu = need_dx or need_gu
        ctx.dims = (T, O, F, K)
        ctx.dtypes = (x.dtype, *(None if p is not None else w.dtype for p, w in zip(packed, (gate_up, down))))
        ctx.whole = packed == (None, None) and need and T > 0 and O > 0
        if ctx.whole:  # one call
            ctx.need = need_dx, need_gu, need_d
            y, gu, saved = _capi.mxfp4_swiglu_train(_matrix(x, "x"), _matrix(gate_up, "gate_up"), _matrix(down, "down"),
                                                    need_dx, need_gu, need_d)
            ctx.save_for_backward(gu if need_dgu else None, saved)
            return y
        if T == 0:
            ctx.save_for_backward(*(None,) * 9)
            return torch.empty((0, O), dtype=torch.bfloat16, device=x.device)
        qx, qxt, _ = _capi.mxfp4_quant(_matrix(x, "x"), rows=True, cols=need_gu)
        qgu, qgut = _weight_codes(wgu, need_dx, "gate_up")
        qd, qdt = _weight_codes(wd, need_dgu, "down")
        gu = qht = None
        if need or F % 128:
            gu = _product(qx, qgu, T, 2 * F, K)
            qh, qht = _capi.mxfp4_swiglu_quant(gu, cols=need_d)
        else:  # activation and h's quantisation in the product's epilogue; gu is not written
            qh = _capi.mxfp4_swiglu_gemm(qx, qgu, T, F, K)
        none = (None, None)
        ctx.save_for_backward(gu if need_dgu else None, *(qxt or none), *(qht or none), *(qgut or none), *(qdt or none))
        return _product(qh, qd, T, O, F)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        T, O, F, K = ctx.dims
        xd, gud, dd = ctx.dtypes
        need_dx, need_gu, need_d = ctx.needs_input_grad[:3]
        dev = dy.device
        if T == 0 or O == 0:
            return (torch.zeros((T, K), dtype=xd, device=dev) if need_dx else None,
                    torch.zeros((2 * F, K), dtype=gud, device=dev) if need_gu else None,
                    torch.zeros((O, F), dtype=dd, device=dev) if need_d else None, None, None)
        if ctx.whole:
            gu, saved = ctx.saved_tensors
            types = (t if n else None for t, n in zip((xd, gud, dd), ctx.need))
            return *_capi.mxfp4_swiglu_bwd(_matrix(dy, "dy"), gu, saved, (T, K, F, O), *types), None, None
        gu, qxt, sxt, qht, sht, qgut, sgut, qdt, sdt = ctx.saved_tensors
        q, qt, _ = _capi.mxfp4_quant(_matrix(dy, "dy"), rows=need_dx or need_gu, cols=need_d)
        dx = dgu = dd_ = None
        if need_d:
            dd_ = _product(qt, (qht, sht), O, F, T, None, dd)
        if need_dx or need_gu:
            dh = _product(q, (qdt, sdt), T, F, O)
            p, pt = _capi.mxfp4_swiglu_bwd_quant(dh, gu, rows=need_dx, cols=need_gu)
            if need_dx:
                dx = _product(p, (qgut, sgut), T, K, 2 * F, None, xd)
            if need_gu:
                dgu = _product(pt, (qxt, sxt), 2 * F, K, T, None, gud)
        return dx, dgu, dd_, None, None


def _split(w, what: str):
    """(tensor for autograd, packed weight) of a weight argument."""
    if isinstance(w, MXFP4Tensor):
        return None, w
    if not isinstance(w, torch.Tensor) or w.dim() != 2 or not w.is_floating_point():
        raise ValueError(f"{what} must be a 2-D floating-point tensor or an MXFP4Tensor")
    return w, None


def _check_input(x: torch.Tensor, k: int, *others) -> torch.Tensor:
    if not isinstance(x, torch.Tensor) or not x.is_floating_point():
        raise ValueError("x must be a floating-point tensor")
    if x.dim() < 1 or x.shape[-1] != k:
        raise ValueError(f"expected input last dim {k}, got {tuple(x.shape)}")
    tensors = [x]
    for o in others:
        if isinstance(o, MXFP4Tensor):
            tensors += [o.codes, o.scales]
        elif o is not None:
            tensors.append(o)
    _capi._require_cuda(*tensors)
    return x if x.dim() == 2 else x.reshape(-1, k)


def mxfp4_linear(x: torch.Tensor, weight: "torch.Tensor | MXFP4Tensor", bias: torch.Tensor | None = None) -> torch.Tensor:
    """``Q(x)·Q(weight)ᵀ (+ bias)`` in bf16: x [..., K], weight [O, K] floating-point (differentiable) or
    ``MXFP4Tensor`` (frozen; the gradient of x needs its transposed form)."""
    w, packed = _split(weight, "weight")
    O, K = weight.shape
    x2 = _check_input(x, K, weight, bias)
    if bias is not None and tuple(bias.shape) != (O,):
        raise ValueError(f"bias must have shape ({O},), got {tuple(bias.shape)}")
    grad = torch.is_grad_enabled() and (x.requires_grad or (w is not None and w.requires_grad)
                                        or (bias is not None and bias.requires_grad))
    if not grad and packed is not None and x2.shape[0] > 0 and not _capi.has_tangent(x, bias):  # (refused by the function)
        y = _capi.mxfp4_linear(_matrix(x2, "x"), packed._pair(), O, K, None if bias is None else _bias(bias, O))
    else:
        y = MXFP4LinearFn.apply(x2, w, bias, packed, grad)
    return y if x.dim() == 2 else y.view(*x.shape[:-1], O)


def mxfp4_swiglu(x: torch.Tensor, gate_up: "torch.Tensor | MXFP4Tensor", down: "torch.Tensor | MXFP4Tensor") -> torch.Tensor:
    """The gated block ``down(silu(g)·u)``, ``[g | u] = x·gate_upᵀ``: x [..., K], gate_up [2F, K] (gate rows, then
    up rows), down [O, F]; F a multiple of 32.  Weights as in ``mxfp4_linear``; the result is bf16."""
    wgu, pgu = _split(gate_up, "gate_up")
    wd, pd = _split(down, "down")
    F2, K = gate_up.shape
    O, F = down.shape
    if F2 != 2 * F or F % 32:
        raise ValueError(f"gated block shapes: gate_up {tuple(gate_up.shape)}, down {tuple(down.shape)} "
                         "(gate_up [2F, K], down [O, F], F a multiple of 32)")
    x2 = _check_input(x, K, gate_up, down)
    grad = torch.is_grad_enabled() and (x.requires_grad or (wgu is not None and wgu.requires_grad)
                                        or (wd is not None and wd.requires_grad))
    if not grad and pgu is not None and pd is not None and F % 128 == 0 and x2.shape[0] > 0 and not _capi.has_tangent(x):
        y = _capi.mxfp4_swiglu_mlp(_matrix(x2, "x"), pgu._pair(), pd._pair(), F, O)
    else:
        y = MXFP4SwiGLUFn.apply(x2, wgu, wd, (pgu, pd), grad)
    return y if x.dim() == 2 else y.view(*x.shape[:-1], O)


class _Frozen(nn.Module):
    """A module whose weights are held in MXFP4 buffers ``<name>_codes`` and ``<name>_scales``."""

    def _hold(self, name: str, q: MXFP4Tensor) -> None:
        self.register_buffer(f"{name}_codes", q.codes)
        self.register_buffer(f"{name}_scales", q.scales)
        t = q.transposed
        self.register_buffer(f"{name}_codes_t", None if t is None else t.codes)
        self.register_buffer(f"{name}_scales_t", None if t is None else t.scales)

    def _held(self, name: str, shape: tuple[int, int]) -> MXFP4Tensor:
        ct = getattr(self, f"{name}_codes_t")
        t = None if ct is None else MXFP4Tensor(ct, getattr(self, f"{name}_scales_t"), (shape[1], shape[0]))
        return MXFP4Tensor(getattr(self, f"{name}_codes"), getattr(self, f"{name}_scales"), shape, t)


def _bitlinear_weight(lin) -> torch.Tensor:
    return lin.int_weight.float() * lin.weight_scale.float()[:, None]


class MXFP4Linear(_Frozen):
    """A frozen linear layer with its weight in MXFP4 (``mxfp4_linear`` on an ``MXFP4Tensor``).

    ``input_grad``: also hold the transposed form, so that gradients pass through to the input."""

    def __init__(self, weight: torch.Tensor, bias: torch.Tensor | None = None, input_grad: bool = False):
        super().__init__()
        q = quantize_fp_to_mxfp4(weight, transposed=input_grad)
        self.out_features, self.in_features = q.shape
        self._hold("weight", q)
        self.register_buffer("bias", None if bias is None else _bias(bias, q.shape[0]).clone())

    @classmethod
    def from_bitlinear(cls, lin, input_grad: bool = False) -> "MXFP4Linear":
        """The layer of a trained ``BitLinear``."""
        return cls(_bitlinear_weight(lin), lin.bias, input_grad)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return mxfp4_linear(x, self._held("weight", (self.out_features, self.in_features)), self.bias)

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}"


class MXFP4SwiGLU(_Frozen):
    """A frozen gated block with its weights in MXFP4 (``mxfp4_swiglu`` on ``MXFP4Tensor`` weights)."""

    def __init__(self, gate_up: torch.Tensor, down: torch.Tensor, input_grad: bool = False):
        super().__init__()
        if gate_up.dim() != 2 or down.dim() != 2 or gate_up.shape[0] != 2 * down.shape[1] or down.shape[1] % 32:
            raise ValueError(f"gated block shapes: gate_up {tuple(gate_up.shape)}, down {tuple(down.shape)}")
        self.d_out, self.ffn = down.shape
        self.d_in = gate_up.shape[1]
        self._hold("gate_up", quantize_fp_to_mxfp4(gate_up, transposed=input_grad))
        self._hold("down", quantize_fp_to_mxfp4(down, transposed=input_grad))

    @classmethod
    def from_swiglu_mlp(cls, mlp, input_grad: bool = False) -> "MXFP4SwiGLU":
        """The block of a trained ``SwiGLUMLP`` (without biases)."""
        if mlp.gate_up.bias is not None or mlp.down.bias is not None:
            raise ValueError("MXFP4SwiGLU holds no biases")
        return cls(_bitlinear_weight(mlp.gate_up), _bitlinear_weight(mlp.down), input_grad)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return mxfp4_swiglu(x, self._held("gate_up", (2 * self.ffn, self.d_in)), self._held("down", (self.d_out, self.ffn)))

    def extra_repr(self) -> str:
        return f"d_in={self.d_in}, ffn={self.ffn}, d_out={self.d_out}"


__all__ = ["MXFP4Tensor", "MXFP4Linear", "MXFP4LinearFn", "MXFP4SwiGLU", "MXFP4SwiGLUFn", "mxfp4_linear",
           "mxfp4_matmul", "mxfp4_swiglu", "quantize_fp_to_mxfp4", "quantize_fp_to_mxfp4_dual"]
