"""Paged-cache writer: append new key rows into a paged KV pool.

The attention path reads its keys from paged pools ``[blocks, block_size, 1,
D]`` through per-batch block tables; this is the step that fills them.  The
layout is the reference's (golden.py:315-360, the inverse of
``unpack_paged_kv``, golden.py:247-268): logical position ``p`` of batch ``b``
lives at ``pool[block_table[b, p // block_size], p % block_size]``.  The
reference has no device writer (its tests pack caches on the host), so this
op has no reference signature; it follows the operator's own conventions
(TND ``cu_seqlens`` for the new rows, int32 tables with -1 = unmapped).

``append_paged_kv`` copies the rows as they are; ``append_paged_kv_norm_rope``
norms and rotates them on the way (``rope.norm_rope`` is the same transform
for the query heads).

Runs ``sas_kv_append`` / ``sas_kv_append_norm_rope`` from ``libsas.so`` on the
caller's stream; there is no CPU fallback.
"""

from __future__ import annotations

import ctypes as C
from typing import Optional

import torch

from . import _lib
from .rope import row_transform


def append_paged_kv(kv_pool: torch.Tensor, block_table: torch.Tensor, new_rows: torch.Tensor,
                    cu_seqlens_new: torch.Tensor, start_pos: torch.Tensor,
                    check_errors: bool = False) -> Optional[list]:
    """Write ``new_rows`` into ``kv_pool`` in place.

    kv_pool:        [blocks, block_size, 1, D] (or [blocks, block_size, D]), bf16/fp16, CUDA.
    block_table:    [B, table_len] int32 (-1 = unmapped page), CUDA.
    new_rows:       [T_new, 1, D] or [T_new, D], same dtype as the pool, CUDA.
    cu_seqlens_new: [B + 1] int32: batch b appends rows cu[b] .. cu[b+1].
    start_pos:      [B] int32: logical position of batch b's first new row
                    (normally its length before the append).

    Rows whose position falls past the table or on an unmapped page are
    skipped.  With ``check_errors`` the call synchronises and returns the
    device error record ``[code, site, row, batch]`` if any row was skipped
    (else None).
    """
    assert kv_pool.is_cuda and new_rows.is_cuda, "kv_pool and new_rows must be CUDA tensors"
    assert kv_pool.dtype == new_rows.dtype, "new_rows must have the pool's dtype"
    assert kv_pool.dim() in (3, 4) and (kv_pool.dim() == 3 or kv_pool.shape[2] == 1), \
        "kv_pool must be [blocks, block_size, 1, D]"
    D = kv_pool.shape[-1]
    assert new_rows.shape[-1] == D, "new_rows last dim must match the pool"
    assert kv_pool.is_contiguous() and new_rows.is_contiguous(), "tensors must be contiguous"
    dev = kv_pool.device
    bt = block_table.to(device=dev, dtype=torch.int32).contiguous()
    cu = cu_seqlens_new.to(device=dev, dtype=torch.int32).contiguous()
    sp = start_pos.to(device=dev, dtype=torch.int32).contiguous()
    B = bt.shape[0]
    assert cu.numel() == B + 1 and sp.numel() == B, "cu_seqlens_new [B+1], start_pos [B]"
    total = new_rows.numel() // D
    err = torch.zeros(4, dtype=torch.int32, device=dev) if check_errors else None
    stream = torch.cuda.current_stream(dev).cuda_stream
    _lib.check("sas_kv_append", _lib.lib().sas_kv_append(
        C.c_void_p(kv_pool.data_ptr()), kv_pool.shape[0], kv_pool.shape[1],
        D * kv_pool.element_size(), C.c_void_p(bt.data_ptr()), bt.shape[1],
        C.c_void_p(new_rows.data_ptr()), C.c_void_p(cu.data_ptr()), C.c_void_p(sp.data_ptr()),
        B, total, C.c_void_p(err.data_ptr() if err is not None else 0), C.c_void_p(stream)))
    if err is not None:
        e = err.tolist()
        return e if e[0] != 0 else None
    return None


def append_paged_kv_norm_rope(kv_pool: torch.Tensor, block_table: torch.Tensor,
                              new_rows: torch.Tensor, cu_seqlens_new: torch.Tensor,
                              start_pos: torch.Tensor, cos: Optional[torch.Tensor] = None,
                              sin: Optional[torch.Tensor] = None, *, norm_dim: int = 0,
                              norm_weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
                              interleaved: bool = True, cmp_ratio: int = 1,
                              check_errors: bool = False) -> Optional[list]:
    """``append_paged_kv`` with each row normed over its first ``norm_dim`` columns and
    its last ``rope_dim`` columns rotated on the way into ``kv_pool``.

    The pool, table, ``cu_seqlens_new`` and ``start_pos`` are ``append_paged_kv``'s; cos,
    sin, norm_dim, norm_weight, eps and interleaved are ``rope.norm_rope``'s.  The row at
    logical position p of its sequence is rotated at position ``p * cmp_ratio`` (the first
    token of those that a row of a ratio-compressed cache stands for).  new_rows
    [T_new, 1, D] or [T_new, D]; rows at or past ``cu_seqlens_new[-1]`` belong to no
    sequence and are left out.

    Rows on an unmapped page or past the tables are skipped; two rows of one call must not
    share a slot.  With ``check_errors`` the call synchronises and returns the device error
    record ``[code, site, row, batch]`` if any row was skipped (else None).
    """
    dev = kv_pool.device
    if dev.type != "cuda" or new_rows.device != dev:
        raise RuntimeError("kv_pool and new_rows must be on one CUDA (sm_100a) device")
    pool_shape = kv_pool.shape
    if len(pool_shape) not in (3, 4) or (len(pool_shape) == 4 and pool_shape[2] != 1):
        raise ValueError("kv_pool must be [blocks, block_size, 1, D]")
    D = pool_shape[-1]
    if new_rows.dtype != kv_pool.dtype or new_rows.shape[-1] != D:
        raise ValueError("new_rows must have the pool's dtype and last dim")
    if not kv_pool.is_contiguous() or not new_rows.is_contiguous():
        raise ValueError("kv_pool and new_rows must be contiguous")
    if pool_shape[1] < 1:
        raise ValueError("block_size must be >= 1")
    table_shape = block_table.shape
    if len(table_shape) != 2 or table_shape[0] < 1:
        raise ValueError("block_table must be [B, table_len] with B >= 1")
    if not 1 <= cmp_ratio <= _lib.INT32_MAX:
        raise ValueError(f"cmp_ratio must be >= 1 (got {cmp_ratio})")
    if max(new_rows.numel() // D, pool_shape[0], pool_shape[1]) > _lib.INT32_MAX:
        raise ValueError("more than 2^31 - 1 rows or blocks")
    B = table_shape[0]
    if cu_seqlens_new.numel() != B + 1 or start_pos.numel() != B:
        raise ValueError("cu_seqlens_new must have B + 1 entries and start_pos B")
    tr = row_transform(kv_pool.dtype, dev, D, cos, sin, int(norm_dim), norm_weight, eps,
                       interleaved, False)
    total = new_rows.numel() // D
    if total == 0:
        return None
    if (kv_pool.data_ptr() | new_rows.data_ptr()) & 15:
        raise ValueError("kv_pool and new_rows must be 16-byte aligned")
    bt = _lib.dev_i32(block_table, dev)
    cu = _lib.dev_i32(cu_seqlens_new, dev)
    sp = _lib.dev_i32(start_pos, dev)
    err = torch.zeros(4, dtype=torch.int32, device=dev) if check_errors else None
    with _lib.on_device(dev) as stream:
        _lib.check("sas_kv_append_norm_rope", _lib.lib().sas_kv_append_norm_rope(
            tr, kv_pool.data_ptr(), pool_shape[0], pool_shape[1], bt.data_ptr(), table_shape[1],
            new_rows.data_ptr(), cu.data_ptr(), sp.data_ptr(), B, total, int(cmp_ratio),
            err.data_ptr() if err is not None else None, stream))
    if err is not None:
        e = err.tolist()
        return e if e[0] != 0 else None
    return None
