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

import ctypes as C
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
    tr = _lib.SasRowTransform(head_dim=head_dim, norm_dim=norm_dim, dtype=code,
                              interleaved=bool(interleaved), inverse=bool(inverse), eps=eps)
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin come together")
    if cos is not None:
        if cos.dim() != 2 or cos.shape != sin.shape:
            raise ValueError("cos and sin must be [positions, rope_dim / 2]")
        rope_dim = 2 * cos.shape[1]
        if rope_dim % 16 or not 16 <= rope_dim <= head_dim:
            raise ValueError(f"rope_dim must be a multiple of 16 up to {head_dim} "
                             f"(got {rope_dim})")
        for name, t in (("cos", cos), ("sin", sin)):
            if t.dtype != torch.float32 or t.device != device or not t.is_contiguous():
                raise ValueError(f"{name} must be a contiguous float32 tensor on {device}")
        tr.cos, tr.sin = cos.data_ptr(), sin.data_ptr()
        tr.table_rows, tr.rope_dim = min(cos.shape[0], 2 ** 31 - 1), rope_dim
    if norm_weight is not None:
        if norm_weight.shape != (norm_dim,):
            raise ValueError(f"norm_weight must be [norm_dim] = [{norm_dim}]")
        if norm_weight.dtype not in (torch.float32, dtype) or norm_weight.device != device \
                or not norm_weight.is_contiguous():
            raise ValueError(f"norm_weight must be contiguous, float32 or {dtype}, on {device}")
        tr.norm_weight = norm_weight.data_ptr() if norm_dim else None
        tr.weight_dtype = _lib.DTYPE_F32 if norm_weight.dtype == torch.float32 else code
    if norm_dim == 0 and cos is None:
        raise ValueError("nothing to do: neither a norm nor a rotation is asked for")
    return tr


def _head_rows(t: torch.Tensor) -> Optional[torch.Tensor]:
    """[T, H, D] view of [..., H, D] that the kernel can address, or None."""
    try:
        v = t.view(-1, t.shape[-2], t.shape[-1])
    except RuntimeError:
        return None
    ok = (v.stride(2) == 1 and v.stride(0) % 8 == 0 and v.stride(1) % 8 == 0
          and v.data_ptr() % 16 == 0)
    return v if ok else None


def _rows_overlap(v: torch.Tensor) -> bool:
    """Whether rows of the [T, H, D] view share memory."""
    end = v.shape[2]
    for stride, size in sorted(zip(v.stride()[:2], v.shape[:2])):
        if size > 1 and stride < end:
            return True
        end = stride * (size - 1) + end
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
    out:         a tensor of x's shape and dtype to write; ``x`` itself works in place,
                 any other overlap does not.

    Rows of a position outside the tables are zeros; with ``check_errors`` the call
    synchronises and raises RuntimeError for them.
    """
    dev = x.device
    if dev.type != "cuda":
        raise RuntimeError(f"norm_rope runs on a CUDA (sm_100a) device only; got x on {dev}")
    if x.dim() not in (3, 4):
        raise ValueError(f"x must be [T, H, D] or [B, S, H, D] (got {tuple(x.shape)})")
    H, D = x.shape[-2], x.shape[-1]
    tr = row_transform(x.dtype, dev, D, cos, sin, int(norm_dim), norm_weight, eps, interleaved,
                       inverse)
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=dev)
    elif out.shape != x.shape or out.dtype != x.dtype or out.device != dev:
        raise ValueError("out must have x's shape, dtype and device")
    T = x.numel() // (H * D) if x.numel() else 0
    pos = None
    if tr.rope_dim:
        if positions is None or positions.dtype not in (torch.int32, torch.int64) \
                or positions.numel() != x.shape[:-2].numel():
            raise ValueError("positions must be int32 or int64 with one entry per token")
        pos = positions.to(dev).contiguous()
    if T == 0:
        return out
    o = _head_rows(out)
    if o is None or _rows_overlap(o):
        raise ValueError("out must have a contiguous last dim, strides of multiples of 8, "
                         "16-byte alignment and rows that do not overlap")
    v = _head_rows(x)
    if v is None:
        v = x.reshape(T, H, D).clone(memory_format=torch.contiguous_format)
    err = torch.zeros(4, dtype=torch.int32, device=dev) if check_errors else None
    with torch.cuda.device(dev):
        _lib.check("sas_norm_rope", _lib.lib().sas_norm_rope(
            C.byref(tr), v.data_ptr(), v.stride(0), v.stride(1), o.data_ptr(), o.stride(0),
            o.stride(1), T, H, pos.data_ptr() if pos is not None else None,
            int(pos is not None and pos.dtype == torch.int64),
            err.data_ptr() if err is not None else None,
            torch.cuda.current_stream(dev).cuda_stream))
    if err is not None:
        e = err.tolist()
        if e[0]:
            raise RuntimeError(f"norm_rope: the position of token {e[2]} is outside the tables")
    return out
