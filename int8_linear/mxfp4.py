"""4-bit linears (MXFP4) for B200 (sm_100a): quantisers and the product.

The operands are microscaled 4-bit floating point: blocks of 32 consecutive values along K,
each value an e2m1 code (0, 0.5, 1, 1.5, 2, 3, 4, 6 with a sign), each block one e8m0
power-of-two scale.  They take a quarter of bf16's bytes and half of int8's, and the tensor
cores multiply them at twice the int8 rate.

    quant_mxfp4(x)                                   -> (q, s)
    add_rmsnorm_quant_mxfp4(x, residual, w, eps)     -> (q, s, residual_out)
    silu_mul_quant_mxfp4(gate_up)                    -> (q, s)
    dequant_mxfp4(q, s, out_dtype)                   -> the values they stand for
    w4a4_mm(a_q, b_q, scale_a, scale_b, out_dtype, bias)

stand beside per_token_quant, add_rmsnorm_quant, silu_mul_quant and w8a8_mm and are called
as those are.  q is uint8 [rows, K/2], the value with the even index in the low nibble.  s
is uint8 [ceil(rows/128), ceil(K/128), 512], the tensor core's own order: the scale of row
r, block b is s[r // 128, b // 4, (r % 32) * 16 + (r // 32) % 4 * 4 + b % 4], the byte 127
standing for 1; bytes of no row or block are 0.  So a weight is quantised once, with
quant_mxfp4, and a slice of 128-row groups of q and s is the operand of those rows.

A block's scale is 2^(floor(log2 max|y|) - 2), the rule of the OCP microscaling format: the
block's largest value lands between 4 and 8 steps and saturates at 6.  Values are rounded to
the nearest, ties to even.  A block that holds an infinity or a NaN becomes NaN.  The
kernels are csrc/mxfp4.cu, csrc/gemm_mxfp4_sm100.cu and csrc/gemv_mxfp4.cu behind the C ABI;
the quantisers and the product are torch custom ops too, under torch.ops.int8_linear.  The
reference package (AshrithaG/int8-linear) has no 4-bit form.
"""

from __future__ import annotations

import ctypes

import torch

from int8_linear import _native
from int8_linear._native import MOST_ROWS, NotSupported
from int8_linear.fused_quant import _ACT, _WEIGHT
from int8_linear.kernel import Config, current_stream

BLOCK = 32
_FLOAT = _WEIGHT  # bf16, fp16 and fp32
_U8 = torch.uint8

__all__ = ["w4a4_mm", "quant_mxfp4", "add_rmsnorm_quant_mxfp4", "silu_mul_quant_mxfp4", "dequant_mxfp4"]


def _rows(x: torch.Tensor, name: str, kinds: dict) -> tuple[int, int, int, int]:
    """(rows, columns, row stride, device index) of a quantiser's input, or the refusal of it."""
    if x.dtype not in kinds:
        raise NotSupported(f"{name} must be one of {[str(k) for k in kinds]}, got {x.dtype}")
    shape, stride = x.shape, x.stride()
    if len(shape) != 2 or (stride[1] != 1 and shape[1] > 1):
        raise NotSupported(f"{name} must be a 2-D tensor with contiguous rows")
    if shape[0] > MOST_ROWS:
        raise NotSupported(f"{name} has {shape[0]} rows, more than {MOST_ROWS}")
    dev = x.get_device()
    if dev < 0:
        raise ValueError(f"the 4-bit quantisers run on a CUDA device, got {x.device}")
    return (*shape, stride[0], dev)


def _matrix(like: torch.Tensor, rows: int, cols: int, dtype: torch.dtype) -> torch.Tensor:
    """An uninitialised matrix on `like`'s device (torch.empty or new_empty with a type takes
    0.5 to 0.9 us more of a call)."""
    return torch.empty_strided((rows, cols), (cols, 1), dtype=dtype, device=like.device)


def _empty(x: torch.Tensor, m: int, k: int) -> tuple[torch.Tensor, torch.Tensor]:
    if k % BLOCK:
        raise NotSupported(f"K={k} must be a multiple of {BLOCK} (whole blocks)")
    q = _matrix(x, m, k >> 1, _U8)
    return q, q.new_empty((m + 127) >> 7, (k + 127) >> 7, 512)


def quant_mxfp4(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(q uint8 [M, K/2], s uint8 [ceil(M/128), ceil(K/128), 512]) of a bf16, fp16 or fp32
    matrix with contiguous rows: an activation (a column slice of a wider matrix is fine,
    no copy is made) or a weight [N, K].  K must be a multiple of 32."""
    m, k, ld, dev = _rows(x, "x", _FLOAT)
    q, s = _empty(x, m, k)
    if m and k:
        _native.on_device(dev, _native.load().i8l_quant_mxfp4, x.data_ptr(), ld, _FLOAT[x.dtype],
                          q.data_ptr(), k >> 1, s.data_ptr(), m, k, current_stream(dev))
    return q, s


def add_rmsnorm_quant_mxfp4(x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor, eps: float):
    """(q, s, residual_out [M, K] or None): fused_quant.add_rmsnorm_quant with its result in
    4 bits.  h = x + residual in float32 (residual_out is h rounded to x's type);
    r = 1 / sqrt(mean(h^2) + eps), computed in float64 and rounded once to float32;
    y = round(round(h * r) * weight), first to the weight's type, then to x's; y is
    block-quantised.  x and residual bf16/fp16 with contiguous rows."""
    m, k, ld, dev = _rows(x, "x", _ACT)
    if weight.dtype not in _WEIGHT or weight.numel() != k or weight.get_device() != dev:
        raise ValueError(f"weight must hold {k} bf16/fp16/fp32 values on {x.device}, got {weight.dtype} "
                         f"{tuple(weight.shape)} on {weight.device}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype
                                 or residual.get_device() != dev or (residual.stride(1) != 1 and k > 1)):
        raise ValueError("residual must match x in shape, dtype and device and have contiguous rows")
    q, s = _empty(x, m, k)
    rout = torch.empty_like(x) if residual is not None else None
    if m and k:
        w = weight if weight.is_contiguous() else weight.contiguous()
        has = residual is not None
        _native.on_device(dev, _native.load().i8l_add_rmsnorm_quant_mxfp4, x.data_ptr(), ld,
                          residual.data_ptr() if has else None, residual.stride(0) if has else 0, w.data_ptr(),
                          _ACT[x.dtype], _WEIGHT[w.dtype], q.data_ptr(), k >> 1, s.data_ptr(),
                          rout.data_ptr() if has else None, k, m, k, eps, current_stream(dev))
    return q, s, rout


def silu_mul_quant_mxfp4(gate_up: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(q, s) of silu(gate) * up for bf16/fp16 rows [gate | up] of 2K values:
    fused_quant.silu_mul_quant with its result in 4 bits.  The product is rounded to
    float32 and then to gate_up's type, as if computed exactly, before the blocks."""
    m, k2, ld, dev = _rows(gate_up, "gate_up", _ACT)
    if k2 % 2:
        raise ValueError(f"gate_up rows of {k2} values are not [gate | up]")
    k = k2 >> 1
    q, s = _empty(gate_up, m, k)
    if m and k:
        _native.on_device(dev, _native.load().i8l_silu_mul_quant_mxfp4, gate_up.data_ptr(), ld,
                          _ACT[gate_up.dtype], q.data_ptr(), k >> 1, s.data_ptr(), m, k, current_stream(dev))
    return q, s


def _scales(s: torch.Tensor, rows: int, k: int, dev: int, name: str) -> torch.Tensor:
    """The scale tiles s of a [rows, k] operand on device `dev`, copied if the kernels cannot
    read them where they lie; raises if they are not that."""
    if s.dtype != _U8:
        raise NotSupported(f"{name} must be uint8 scale bytes, got {s.dtype}")
    if s.shape != ((rows + 127) >> 7, (k + 127) >> 7, 512) or s.get_device() != dev:
        raise ValueError(f"{name} must be the {[-(-rows // 128), -(-k // 128), 512]} scale tiles of [{rows}, {k}] on "
                         f"device {dev}, got {tuple(s.shape)} on {s.device}")
    if s.is_contiguous() and s.data_ptr() % 16 == 0:
        return s
    return _copied(s, name)


def _copied(t: torch.Tensor, name: str) -> torch.Tensor:
    """A contiguous copy.  A kernel launched programmatically reads weights before the copy
    must have finished, so a weight that needs one is refused then."""
    if name in ("b_q", "scale_b") and _native.pdl_enabled():
        raise NotSupported(f"with programmatic dependent launch {name} must be 16-byte aligned and contiguous")
    return t.clone(memory_format=torch.contiguous_format)


def dequant_mxfp4(q: torch.Tensor, s: torch.Tensor, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """[M, K] values that codes q [M, K/2] and scales s stand for, in bf16, fp16 or fp32."""
    if q.dtype != _U8 or out_dtype not in _FLOAT:
        raise NotSupported(f"uint8 codes to bf16, fp16 or fp32 only, got {q.dtype} to {out_dtype}")
    shape, stride = q.shape, q.stride()
    if len(shape) != 2 or (stride[1] != 1 and shape[1] > 1):
        raise NotSupported("q must be a 2-D tensor with contiguous rows")
    m, half = shape
    k, dev, ldq = 2 * half, q.get_device(), stride[0]
    if k % BLOCK or m > MOST_ROWS:
        raise NotSupported(f"K={k} must be a multiple of {BLOCK} (whole blocks) and M={m} at most {MOST_ROWS}")
    if dev < 0:
        raise ValueError(f"dequant_mxfp4 runs on a CUDA device, got {q.device}")
    s = _scales(s, m, k, dev, "s")
    out = _matrix(q, m, k, out_dtype)
    if m and k:
        if q.data_ptr() % 4 or ldq % 4 or ldq < half:
            q, ldq = q.clone(memory_format=torch.contiguous_format), half
        _native.on_device(dev, _native.load().i8l_dequant_mxfp4, q.data_ptr(), ldq, s.data_ptr(),
                          out.data_ptr(), k, _FLOAT[out_dtype], m, k, current_stream(dev))
    return out


SPLIT_TILES = (16, 32, 64, 128)


def _tile(config: Config) -> _native.I8LTile:
    """The C tile of a Config for the 4-bit product: swap_ab token tiles with split 0, 1 or 3,
    CTA pairs (split 4) or CUDA cores (split 5)."""
    if config.split == 5 and config.bm in (1, 2, 4) and config.bn == 0:
        return _native.I8LTile(tok_tile=config.bm, split=5)
    if config.split == 4 and not config.swapped and config.bm == 128 and config.bn == 256:
        return _native.I8LTile(tok_tile=128, w_tile=256, stages=config.stages, ctas=config.ctas, split=4)
    if config.split not in (0, 1, 3) or not config.swapped or config.bm not in SPLIT_TILES or config.bn != 128:
        raise NotSupported(f"{config.name}: 4-bit tiles are bm in {SPLIT_TILES} x bn 128 with swap_ab, pairs "
                           "(128 x 256, split 4) or CUDA cores (bm 1, 2 or 4, bn 0, split 5)")
    return _native.I8LTile(swap_ab=1, tok_tile=config.bm, w_tile=128, stages=config.stages, split=config.split,
                           cluster=1 if config.split == 1 else config.cluster)


def w4a4_mm(a_q: torch.Tensor, b_q: torch.Tensor, scale_a: torch.Tensor, scale_b: torch.Tensor,
            out_dtype: torch.dtype = torch.bfloat16, bias: torch.Tensor | None = None, *,
            config: Config | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """A @ W^T + bias [M, N] for 4-bit A [M, K] and W [N, K].

    As w8a8_mm, with 4-bit operands: a_q is [M, K/2] codes, b_q the transposed view
    [K/2, N] of a weight's [N, K/2] codes (`w_q.t()`), scale_a and scale_b their scale tiles
    as quant_mxfp4 gives them.  The sum is float32 on the tensor cores, bias (bf16, fp16 or
    fp32, [N]) is added in float32, and one rounding makes the bf16, fp16 or fp32 output.
    `out` is an [M, N] tensor with contiguous rows to write into.  `config` picks a tiling
    (swap_ab token tiles of 16 to 128 with split 1 or 3, cluster and stages; CTA pairs: bm
    128, bn 256, split 4; or CUDA cores for at most four tokens: bm 1, 2 or 4, bn 0, split 5)
    in place of the library's choice.  Raises NotSupported for what the kernel does not take and ValueError
    for inconsistent arguments.  With programmatic dependent launch (set_pdl) a weight
    that quant_mxfp4 did not make, with it on, must be complete before the call: the stream
    synchronised, or a kernel of another library launched, after whatever wrote it."""
    if a_q.dtype != _U8 or b_q.dtype != _U8:
        raise NotSupported(f"uint8 4-bit codes only, got {a_q.dtype} and {b_q.dtype}")
    shape_a, shape_b = a_q.shape, b_q.shape
    if len(shape_a) != 2 or len(shape_b) != 2 or shape_a[1] != shape_b[0]:
        raise ValueError(f"cannot multiply {tuple(shape_a)} by {tuple(shape_b)}")
    m, half = shape_a
    n, k, dev = shape_b[1], 2 * half, a_q.get_device()
    if k == 0 or k % BLOCK or m > MOST_ROWS or n > MOST_ROWS:
        raise NotSupported(f"K={k} must be a positive multiple of {BLOCK} (whole blocks), M={m} and N={n} at most "
                           f"{MOST_ROWS}")
    lda, unit_a = a_q.stride()
    unit_b, ldw = b_q.stride()
    if unit_b != 1 and n > 1:
        raise NotSupported("b_q must be the K-contiguous [K/2, N] view of an [N, K/2] weight")
    if dev < 0 or b_q.get_device() != dev:
        raise ValueError(f"w4a4_mm runs on one CUDA device; got tensors on {a_q.device} and {b_q.device}")
    sa, sb = _scales(scale_a, m, k, dev, "scale_a"), _scales(scale_b, n, k, dev, "scale_b")
    bias_ptr, bias_code = None, 0
    if bias is not None:
        if bias.shape != (n,) or bias.get_device() != dev:
            raise ValueError(f"bias must have shape ({n},) on {a_q.device}, got {tuple(bias.shape)} on {bias.device}")
        if bias.dtype not in _FLOAT:
            raise NotSupported(f"bias dtype {bias.dtype} not supported")
        bias = bias if bias.is_contiguous() else bias.contiguous()
        bias_ptr, bias_code = bias.data_ptr(), _FLOAT[bias.dtype]
    if out_dtype not in _FLOAT:
        raise NotSupported(f"output dtype {out_dtype} not supported")
    ldc = n
    if out is None:
        out = _matrix(a_q, m, n, out_dtype)
    elif out.shape != (m, n) or out.dtype != out_dtype or out.get_device() != dev \
            or (out.stride(1) != 1 and n > 1):
        raise ValueError(f"out must be a {out_dtype} [{m}, {n}] tensor with contiguous rows on "
                         f"{a_q.device}, got {out.dtype} {tuple(out.shape)} strides {out.stride()}")
    elif m > 1:
        ldc = out.stride(0)
    tile = ctypes.byref(_tile(config)) if config is not None else None
    if m == 0 or n == 0:
        return out
    # TMA reads rows that start on 16-byte boundaries; others are copied.
    ap, wp = a_q.data_ptr(), b_q.data_ptr()
    if ap % 16 or lda % 16 or lda < half or unit_a != 1:
        a_q = a_q.clone(memory_format=torch.contiguous_format)
        ap, lda = a_q.data_ptr(), half
    if wp % 16 or ldw % 16 or ldw < half or unit_b != 1:
        w = _copied(b_q.t(), "b_q")
        wp, ldw = w.data_ptr(), half
    _native.on_device(dev, _native.load().i8l_w4a4_mm, ap, lda, sa.data_ptr(), wp, ldw, sb.data_ptr(), bias_ptr,
                      bias_code, out.data_ptr(), _FLOAT[out_dtype], ldc, m, n, k, tile, current_stream(dev))
    return out


@torch.library.custom_op("int8_linear::quant_mxfp4", mutates_args=())
def quant_mxfp4_op(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    return quant_mxfp4(x.contiguous())


def _fake(x, m, k):
    return (x.new_empty((m, k // 2), dtype=torch.uint8),
            x.new_empty(((m + 127) // 128, (k + 127) // 128, 512), dtype=torch.uint8))


@quant_mxfp4_op.register_fake
def _(x):
    return _fake(x, x.shape[0], x.shape[1])


@torch.library.custom_op("int8_linear::rmsnorm_quant_mxfp4", mutates_args=())
def rmsnorm_quant_mxfp4_op(x: torch.Tensor, weight: torch.Tensor, eps: float) -> tuple[torch.Tensor, torch.Tensor]:
    q, s, _ = add_rmsnorm_quant_mxfp4(x.contiguous(), None, weight, eps)
    return q, s


@rmsnorm_quant_mxfp4_op.register_fake
def _(x, weight, eps):
    return _fake(x, x.shape[0], x.shape[1])


@torch.library.custom_op("int8_linear::add_rmsnorm_quant_mxfp4", mutates_args=())
def add_rmsnorm_quant_mxfp4_op(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor,
                               eps: float) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    return add_rmsnorm_quant_mxfp4(x.contiguous(), residual.contiguous(), weight, eps)


@add_rmsnorm_quant_mxfp4_op.register_fake
def _(x, residual, weight, eps):
    return (*_fake(x, x.shape[0], x.shape[1]), x.new_empty(x.shape))


@torch.library.custom_op("int8_linear::silu_mul_quant_mxfp4", mutates_args=())
def silu_mul_quant_mxfp4_op(gate_up: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    return silu_mul_quant_mxfp4(gate_up.contiguous())


@silu_mul_quant_mxfp4_op.register_fake
def _(gate_up):
    return _fake(gate_up, gate_up.shape[0], gate_up.shape[1] // 2)


@torch.library.custom_op("int8_linear::w4a4_mm", mutates_args=())
def w4a4_mm_op(a_q: torch.Tensor, b_q: torch.Tensor, scale_a: torch.Tensor, scale_b: torch.Tensor,
               out_dtype: torch.dtype, bias: torch.Tensor | None) -> torch.Tensor:
    return w4a4_mm(a_q, b_q, scale_a, scale_b, out_dtype, bias)


@w4a4_mm_op.register_fake
def _(a_q, b_q, scale_a, scale_b, out_dtype, bias):
    return a_q.new_empty((a_q.shape[0], b_q.shape[1]), dtype=out_dtype)
