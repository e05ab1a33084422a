"""RMSNorm of every query and key head with the position rotation in the same pass, on
B200 (sm_100a).

    qk_norm_rope(qkv, q_weight, k_weight, eps, positions, cos_sin, heads, kv_heads) -> (q, k)

is the step between the qkv linear of a Qwen3-shaped layer and its attention: each head is
normalised over its own values, scaled by its weight and rotated by its token's position.
The kernel is csrc/qk_norm.cu behind the C ABI; float32 inside, with a power of two taken out
of bf16 heads whose squares float32 cannot hold, and one rounding at the end; also
torch.ops.int8_linear.qk_norm_rope.
The reference package (AshrithaG/int8-linear) leaves this step to vLLM.
"""

from __future__ import annotations

import torch

from int8_linear import _native
from int8_linear._native import MOST_ROWS, NotSupported
from int8_linear.fused_quant import _ACT, _WEIGHT
from int8_linear.kernel import current_stream

__all__ = ["qk_norm_rope"]


def _out(out: torch.Tensor | None, shape: tuple, like: torch.Tensor, name: str) -> torch.Tensor:
    if out is None:
        return like.new_empty(*shape)  # a tuple takes 0.4 us more
    if out.shape != shape or out.dtype != like.dtype or out.get_device() != like.get_device() \
            or out.stride(2) != 1 or out.stride(1) != shape[2]:
        raise ValueError(f"{name} must be a {like.dtype} {list(shape)} tensor on {like.device} whose heads "
                         f"follow one another, got {out.dtype} {tuple(out.shape)} strides {out.stride()}")
    return out


def qk_norm_rope(qkv: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor, eps: float,
                 positions: torch.Tensor, cos_sin: torch.Tensor, heads: int, kv_heads: int, *,
                 interleaved: bool = False, q_out: torch.Tensor | None = None,
                 k_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """(q [M, heads, D], k [M, kv_heads, D]) of a bf16/fp16 qkv [M, >= (heads + kv_heads) D].

    A row of qkv holds the query heads, then the key heads; what follows is left alone.
    For each head, n = x / sqrt(mean(x^2) + eps) * weight, then the first R values of n
    are rotated in pairs (a, b) -> (a cos - b sin, b cos + a sin).  D is the weights'
    length; `positions` [M] (int32 or int64) picks the rows of `cos_sin` [positions, R],
    R/2 cosines followed by R/2 sines (bf16, fp16 or fp32).  Pair i is (n[i], n[i + R/2]),
    or (n[2i], n[2i + 1]) with `interleaved`.  A token whose position is not a row of
    cos_sin comes out as NaN.

    `q_out` and `k_out` are [M, heads, D] tensors to write into, any distance between
    tokens; they may be the heads' own places in qkv
    (`qkv[:, :heads * D].view(M, heads, D)`), but overlap it in no other way.

    Takes D a multiple of 8 up to 256, R a multiple of 16 (8 with interleaved) up to D and
    16-byte aligned rows; raises NotSupported for others, ValueError for inconsistent
    arguments.  R = 0 only normalises."""
    if qkv.dtype not in _ACT:
        raise NotSupported(f"activations must be bfloat16 or float16, got {qkv.dtype}")
    shape, stride = qkv.shape, qkv.stride()
    if len(shape) != 2 or (stride[1] != 1 and shape[1] > 1):
        raise NotSupported("qkv must be a 2-D activation with contiguous rows")
    m, width = shape
    if m > MOST_ROWS:
        raise NotSupported(f"{m} tokens are more than {MOST_ROWS}")
    d, dev = q_weight.numel(), qkv.get_device()
    wdt = q_weight.dtype
    if wdt not in _WEIGHT or k_weight.dtype != wdt or k_weight.numel() != d or d == 0:
        raise ValueError(f"q_weight and k_weight must hold one head's values in one bf16/fp16/fp32 type, got "
                         f"{q_weight.dtype} {tuple(q_weight.shape)} and {k_weight.dtype} {tuple(k_weight.shape)}")
    if heads < 0 or kv_heads < 0 or width < (heads + kv_heads) * d:
        raise ValueError(f"qkv rows of {width} values do not hold {heads} + {kv_heads} heads of {d}")
    wide = positions.dtype == torch.int64
    if not (wide or positions.dtype == torch.int32) or positions.shape != (m,):
        raise ValueError(f"positions must be {m} int32 or int64 values, got {positions.dtype} "
                         f"{tuple(positions.shape)}")
    angles = cos_sin.shape
    if len(angles) != 2 or cos_sin.dtype not in _WEIGHT or angles[1] > d or angles[1] % 2:
        raise ValueError(f"cos_sin must be a bf16/fp16/fp32 [positions, even rot <= {d}] table, got "
                         f"{cos_sin.dtype} {tuple(cos_sin.shape)}")
    if dev < 0:
        raise ValueError(f"qk_norm_rope runs on a CUDA device, got {qkv.device}")
    if not (q_weight.get_device() == k_weight.get_device() == positions.get_device() == cos_sin.get_device() == dev):
        raise ValueError(f"the weights, positions and cos_sin must be on {qkv.device}")
    q = _out(q_out, (m, heads, d), qkv, "q_out")
    k = _out(k_out, (m, kv_heads, d), qkv, "k_out")
    if m == 0 or heads + kv_heads == 0:
        return q, k
    wq = q_weight if q_weight.is_contiguous() else q_weight.contiguous()
    wk = k_weight if k_weight.is_contiguous() else k_weight.contiguous()
    pos = positions if positions.is_contiguous() else positions.contiguous()
    table = cos_sin if cos_sin.is_contiguous() else cos_sin.contiguous()
    length, rot = angles
    _native.on_device(dev, _native.load().i8l_qk_norm_rope, qkv.data_ptr(), stride[0], _ACT[qkv.dtype],
                      wq.data_ptr(), wk.data_ptr(), _WEIGHT[wdt], eps, pos.data_ptr(), wide, table.data_ptr(),
                      _WEIGHT[table.dtype], length, q.data_ptr(), q.stride(0) if m > 1 else 0, k.data_ptr(),
                      k.stride(0) if m > 1 else 0, m, heads, kv_heads, d, rot, interleaved, current_stream(dev))
    return q, k


@torch.library.custom_op("int8_linear::qk_norm_rope", mutates_args=())
def qk_norm_rope_op(qkv: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor, eps: float,
                    positions: torch.Tensor, cos_sin: torch.Tensor, heads: int, kv_heads: int,
                    interleaved: bool) -> tuple[torch.Tensor, torch.Tensor]:
    return qk_norm_rope(qkv, q_weight, k_weight, eps, positions, cos_sin, heads, kv_heads, interleaved=interleaved)


@qk_norm_rope_op.register_fake
def _(qkv, q_weight, k_weight, eps, positions, cos_sin, heads, kv_heads, interleaved):
    m, d = qkv.shape[0], q_weight.numel()
    return qkv.new_empty((m, heads, d)), qkv.new_empty((m, kv_heads, d))
