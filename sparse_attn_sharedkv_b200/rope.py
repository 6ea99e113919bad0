"""Norm and rotation of query (or key) heads in one pass.

The attention takes ``q`` with its norm and its position rotation applied
(the reference does, api.py:129-153: it has no such step).  ``norm_rope``
makes that ``q`` from a projection's output: for each head row, the first
``norm_dim`` columns are normed (root mean square) and the last ``rope_dim``
columns, the ones behind the shared latent, are rotated by the angles of the
token's position.  ``inverse`` turns the other way (an attention output whose
values carried the rotation).  ``kv_cache.append_paged_kv_norm_rope`` is the
same transform for the key rows on their way into the cache.

Runs ``sas_norm_rope`` from ``libsas.so`` on the caller's stream; there is no
CPU fallback and no backward pass.
"""

from __future__ import annotations

from typing import Optional

import torch

from . import _lib

_ROW_DTYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_FP16}


def row_transform(dtype, device, head_dim, cos, sin, norm_dim, norm_weight, eps, interleaved,
                  inverse) -> _lib.SasRowTransform:
    """Check the arguments of the transform and fill its C struct (which
    borrows the tensors: the caller keeps them alive over the call)."""
    code = _ROW_DTYPES.get(dtype)
    if code is None:
        raise ValueError(f"rows must be bfloat16 or float16 (got {dtype})")
    if head_dim % 8 or not 8 <= head_dim <= _lib.SAS_MAX_ROW_DIM:
        raise ValueError(f"head dim must be a multiple of 8 up to {_lib.SAS_MAX_ROW_DIM} "
                         f"(got {head_dim})")
    if norm_dim % 8 or not 0 <= norm_dim <= head_dim:
        raise ValueError(f"norm_dim must be a multiple of 8 in [0, {head_dim}] (got {norm_dim})")
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin come together")
    cos_ptr = sin_ptr = weight_ptr = None
    rows = rope_dim = weight_code = 0
    if cos is not None:
        shape = cos.shape
        if len(shape) != 2 or shape != sin.shape:
            raise ValueError("cos and sin must be [positions, rope_dim / 2]")
        rows, rope_dim = min(shape[0], _lib.INT32_MAX), 2 * shape[1]
        if rows < 1:
            raise ValueError("cos and sin hold no position")
        if rope_dim % 16 or not 16 <= rope_dim <= min(head_dim, _lib.SAS_MAX_ROPE_DIM):
            raise ValueError(f"rope_dim must be a multiple of 16 up to "
                             f"{min(head_dim, _lib.SAS_MAX_ROPE_DIM)} (got {rope_dim})")
        for name, t in (("cos", cos), ("sin", sin)):
            if t.dtype is not torch.float32 or t.device != device or not t.is_contiguous():
                raise ValueError(f"{name} must be a contiguous float32 tensor on {device}")
        cos_ptr, sin_ptr = cos.data_ptr(), sin.data_ptr()
        if (cos_ptr | sin_ptr) & 15:
            raise ValueError("cos and sin must be 16-byte aligned")
    if norm_weight is not None:
        if norm_weight.shape != (norm_dim,):
            raise ValueError(f"norm_weight must be [norm_dim] = [{norm_dim}]")
        wt = norm_weight.dtype
        if (wt is not torch.float32 and wt is not dtype) or norm_weight.device != device \
                or not norm_weight.is_contiguous():
            raise ValueError(f"norm_weight must be contiguous, float32 or {dtype}, on {device}")
        if norm_dim:
            weight_ptr = norm_weight.data_ptr()
            if weight_ptr & 15:
                raise ValueError("norm_weight must be 16-byte aligned")
        weight_code = _lib.DTYPE_F32 if wt is torch.float32 else code
    if norm_dim == 0 and cos is None:
        raise ValueError("nothing to do: neither a norm nor a rotation is asked for")
    if norm_dim and not eps >= 0:
        raise ValueError(f"eps must not be negative (got {eps})")
    return _lib.SasRowTransform(cos_ptr, sin_ptr, weight_ptr, rows, head_dim, norm_dim, rope_dim,
                                code, weight_code, bool(interleaved), bool(inverse), eps)


def _head_rows(t: torch.Tensor):
    """(data pointer, token stride, head stride) by which the kernel can
    address [..., H, D] ``t`` as [T, H, D], or None."""
    if t.dim() == 4:
        try:
            t = t.view(-1, t.shape[-2], t.shape[-1])
        except RuntimeError:
            return None
    st, sh, sd = t.stride()
    ptr = t.data_ptr()
    return (ptr, st, sh) if sd == 1 and not (st | sh) & 7 and not ptr & 15 else None


def _rows_overlap(sizes, strides, width: int) -> bool:
    """Whether rows of ``width`` elements at these sizes and strides share memory."""
    end = width
    for stride, size in sorted(zip(strides, sizes)):
        if size > 1 and stride < end:
            return True
        end += stride * (size - 1)
    return False


def norm_rope(x: torch.Tensor, positions: Optional[torch.Tensor] = None,
              cos: Optional[torch.Tensor] = None, sin: Optional[torch.Tensor] = None, *,
              norm_dim: int = 0, norm_weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
              interleaved: bool = True, inverse: bool = False,
              out: Optional[torch.Tensor] = None, check_errors: bool = False) -> torch.Tensor:
    """Norm and rotate the heads of ``x``; returns ``out`` (new unless given).

    x:           [T, H, D] (TND) or [B, S, H, D] (BSND), bf16 / fp16, CUDA.  Strided
                 views are read in place where the last dim is contiguous and the
                 others are multiples of 8 elements.
    positions:   int32 / int64, one per token ([T] or [B, S]).
    cos, sin:    float32 [positions, rope_dim / 2] tables; the last rope_dim columns are
                 rotated, as pairs (2 i, 2 i + 1) or, with ``interleaved=False``,
                 (i, i + rope_dim / 2).  None: no rotation.
    norm_dim:    columns, from the first, that are normed together (0: no norm);
                 ``norm_weight`` [norm_dim] float32 or x's dtype, None for ones.
    inverse:     rotate by the negative angles.
    out:         a tensor of x's shape and dtype to write: the last dim contiguous, the
                 others multiples of 8 elements, B and S one stride apart, 16-byte aligned.
                 ``x`` itself works in place, any other overlap does not.

    Rows of a position outside the tables are zeros; with ``check_errors`` the call
    synchronises and raises RuntimeError for them.
    """
    dev = x.device
    if dev.type != "cuda":
        raise RuntimeError(f"norm_rope runs on a CUDA (sm_100a) device only; got x on {dev}")
    shape = x.shape
    if len(shape) not in (3, 4):
        raise ValueError(f"x must be [T, H, D] or [B, S, H, D] (got {tuple(shape)})")
    H, D = shape[-2], shape[-1]
    tr = row_transform(x.dtype, dev, D, cos, sin, int(norm_dim), norm_weight, eps, interleaved,
                       inverse)
    T = shape[0] if len(shape) == 3 else shape[0] * shape[1]
    if T * H > 2 ** 31 - 1:
        raise ValueError("x holds more than 2^31 - 1 rows")
    pos_ptr, pos64 = None, 0
    if cos is not None:
        if positions is None or positions.dtype not in (torch.int32, torch.int64) \
                or positions.numel() != T:
            raise ValueError("positions must be int32 or int64 with one entry per token")
        if positions.device != dev or not positions.is_contiguous():
            positions = positions.to(dev).contiguous()
        pos_ptr, pos64 = positions.data_ptr(), positions.dtype is torch.int64
    if out is None:
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
        o = (out.data_ptr(), H * D, D)
    else:
        if out.shape != shape or out.dtype != x.dtype or out.device != dev:
            raise ValueError("out must have x's shape, dtype and device")
        o = _head_rows(out)
        if T * H > 0 and (o is None or _rows_overlap((T, H), o[1:], D)):
            raise ValueError("out must have a contiguous last dim, strides of multiples of 8, "
                             "16-byte alignment and rows that do not overlap")
    if T * H == 0:
        return out
    v = _head_rows(x)
    if v is None:
        x = x.clone(memory_format=torch.contiguous_format)
        v = (x.data_ptr(), H * D, D)
    err = torch.zeros(4, dtype=torch.int32, device=dev) if check_errors else None
    with _lib.on_device(dev) as stream:
        _lib.check("sas_norm_rope", _lib.lib().sas_norm_rope(
            tr, *v, *o, T, H, pos_ptr, pos64, err.data_ptr() if err is not None else None,
            stream))
    if err is not None:
        e = err.tolist()
        if e[0]:
            raise RuntimeError(f"norm_rope: the position of token {e[2]} is outside the tables")
    return out
