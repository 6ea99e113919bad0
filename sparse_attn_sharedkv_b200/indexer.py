"""Selection of the key positions the top-k attention reads.

The attention takes ``cmp_sparse_indices`` (scenario SCFA, api.py:129-153);
this module makes them.  Each token scores the keys of its sequence with
narrow index heads against a paged cache of index keys,

    score[t, j] = sum_h weights[t, h] * relu(q[t, h, :] . key[j, :]),

over the positions the causal threshold leaves it (golden.py:48-62: j <
(seqused_kv - q_len + s + 1) // cmp_ratio), and keeps the positions of the
``topk`` largest.  One index key stands for ``cmp_ratio`` tokens, as one row of
the compressed cache does.

* ``index_scores``: the scores, float32, -inf where a token sees no key.
* ``select_topk``: positions of the largest scores of each row.
* ``select_keys``: both, in a workspace of bounded size.

Runs ``sas_index_scores`` / ``sas_topk_select`` from ``libsas.so`` on the
caller's stream; lengths are read on the device only, so the calls can be
captured in a CUDA graph.  No CPU fallback, no backward pass.
"""

from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from . import _lib
from .api import _check_device_errors, _dtype_code

# Bytes of scores that select_keys holds at a time.  Fewer launches, and their tails,
# gain more than scores that are still in L2: 8 x 4096 causal tokens take 1.27 ms so
# (in the same run their scores 1.10 ms and the selection 0.17 ms), 1.32 ms with 64 MiB,
# 1.59 ms with 16 MiB and 1.25 ms with all 512 MiB.
_SCORE_WORKSPACE = 256 << 20


def _index_params(q, weights, key_pool, block_table, cu_seqlens_q, seqused_kv, cmp_ratio, layout_q,
                  max_keys):
    """Validate the arguments; returns the C struct (without outputs), the
    number of columns and the tensors the struct points to."""
    code = _dtype_code(q.dtype)
    dev, shape = q.device, q.shape
    if dev.type != "cuda":
        raise RuntimeError(f"index scores run on a CUDA (sm_100a) device only; got q on {dev}")
    if layout_q == "TND":
        if len(shape) != 3:
            raise ValueError(f"q must be [T, H, D] in TND (got {tuple(shape)})")
        if cu_seqlens_q is None:
            raise ValueError("cu_seqlens_q is required for TND")
        total, S, B = shape[0], 0, cu_seqlens_q.numel() - 1
    elif layout_q == "BSND":
        if len(shape) != 4:
            raise ValueError(f"q must be [B, S, H, D] in BSND (got {tuple(shape)})")
        B, S = shape[0], shape[1]
        total = B * S
        if cu_seqlens_q is not None and cu_seqlens_q.numel() != B + 1:
            raise ValueError("cu_seqlens_q must have B + 1 entries")
    else:
        raise ValueError(f"unsupported layout_q={layout_q!r}")
    H, D = shape[-2], shape[-1]
    if not 1 <= H <= _lib.SAS_MAX_INDEX_HEADS:
        raise ValueError(f"index heads must be in [1, {_lib.SAS_MAX_INDEX_HEADS}] (got {H})")
    if D % 8 or not 8 <= D <= _lib.SAS_MAX_INDEX_DIM:
        raise ValueError(f"index head dim must be a multiple of 8 up to "
                         f"{_lib.SAS_MAX_INDEX_DIM} (got {D})")
    if B < 1 and total > 0:
        raise ValueError("at least one sequence is needed")
    if weights.shape != shape[:-1] or weights.dtype is not torch.float32:
        raise ValueError("weights must be float32 of q's shape without the last dim")
    pool_shape = key_pool.shape
    if len(pool_shape) not in (3, 4) or (len(pool_shape) == 4 and pool_shape[2] != 1):
        raise ValueError("key_pool must be [blocks, block_size, 1, D]")
    if pool_shape[-1] != D or key_pool.dtype is not q.dtype:
        raise ValueError("q and key_pool must share the head dim and the dtype")
    if pool_shape[1] < 1:
        raise ValueError("block_size must be >= 1")
    if pool_shape[0] * pool_shape[1] > 2 ** 31 - 2:
        raise ValueError("key_pool holds more than 2^31 - 2 rows")
    table_shape = block_table.shape
    if len(table_shape) != 2 or table_shape[0] < B:
        raise ValueError("block_table must be [B, table_len]")
    if seqused_kv.numel() < B:
        raise ValueError("seqused_kv must have one entry per sequence")
    if weights.device != dev or key_pool.device != dev:
        raise ValueError("weights and key_pool must be on q's device")
    if not 1 <= cmp_ratio <= _lib.INT32_MAX:
        raise ValueError(f"cmp_ratio must be >= 1 (got {cmp_ratio})")
    if total > _lib.INT32_MAX:
        raise ValueError(f"q holds more than 2^31 - 1 tokens ({total})")
    N = table_shape[1] * pool_shape[1] if max_keys is None else int(max_keys)
    if not 0 <= N <= _lib.INT32_MAX - 65536:
        raise ValueError(f"max_keys out of range ({N})")
    qf, w, pool = q.contiguous(), weights.contiguous(), key_pool.contiguous()
    if (qf.data_ptr() | pool.data_ptr()) & 15:
        raise ValueError("q and key_pool must be 16-byte aligned")
    bt, kv = _lib.dev_i32(block_table, dev), _lib.dev_i32(seqused_kv, dev)
    cu = _lib.dev_i32(cu_seqlens_q, dev) if cu_seqlens_q is not None else None
    p = _lib.SasIndexParams(
        qf.data_ptr(), w.data_ptr(), pool.data_ptr(), bt.data_ptr(),
        cu.data_ptr() if cu is not None else None, kv.data_ptr(), None, None, None, B, total, S, H,
        D, code, pool_shape[1], pool_shape[0], table_shape[1], int(cmp_ratio), N)
    return p, N, (qf, w, pool, bt, kv, cu)


def _raise_device_error(err) -> None:
    e = err.tolist()
    if e[0]:
        raise RuntimeError(f"sas_index_scores device check failed: code={e[0]} site={e[1]} "
                           f"detail={e[2]} {e[3]}")


def index_scores(q: torch.Tensor, weights: torch.Tensor, *, key_pool: torch.Tensor,
                 block_table: torch.Tensor, cu_seqlens_q: Optional[torch.Tensor] = None,
                 seqused_kv: torch.Tensor, cmp_ratio: int = 1, layout_q: str = "TND",
                 max_keys: Optional[int] = None, return_lengths: bool = False
                 ) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Index scores of each token against the keys of its sequence.

    q:            [T, H, D] (TND, with cu_seqlens_q [B + 1]: tokens before its first and at
                  or past its last entry see no key) or [B, S, H, D] (BSND; tokens past a
                  given q_len see no key), bf16 / fp16, H in 1..128, D a multiple of 8 up to
                  128.
    weights:      float32 [T, H] / [B, S, H]; any softmax or width scale is folded in.
    key_pool:     [blocks, block_size, 1, D] index keys, q's dtype; block_table
                  [B, table_len] int32.  A position whose page is -1 or past the table
                  scores -inf.
    seqused_kv:   [B] uncompressed lengths, the new tokens included.
    max_keys:     columns of the result; positions at and past it are not scored.
                  Default: table_len * block_size.

    Returns float32 scores [T, N] / [B, S, N], -inf at the positions a token does not see
    (rows may be strided), and with ``return_lengths`` also int32 [T] / [B, S]: how many
    positions each token sees.
    """
    p, N, keep = _index_params(q, weights, key_pool, block_table, cu_seqlens_q, seqused_kv,
                               cmp_ratio, layout_q, max_keys)
    dev, total = q.device, p.total_tokens
    # Rows of whole 16-byte vectors.
    stride = (N + 3) // 4 * 4
    scores = weights.new_empty((total, stride))
    if stride != N:
        scores = scores[:, :N]
    lengths = torch.empty(total, dtype=torch.int32, device=dev) if return_lengths else None
    if total > 0:
        err = torch.zeros(4, dtype=torch.int32, device=dev) if _check_device_errors() else None
        p.scores, p.score_stride = scores.data_ptr(), stride
        p.lengths = lengths.data_ptr() if lengths is not None else None
        p.err = err.data_ptr() if err is not None else None
        p.first_token, p.num_tokens, p.fill = 0, total, 1
        with _lib.on_device(dev) as stream:
            _lib.check("sas_index_scores", _lib.lib().sas_index_scores(p, stream))
        if err is not None:
            _raise_device_error(err)
    del keep
    if layout_q == "BSND":
        scores = scores.unflatten(0, q.shape[:2])
        lengths = lengths.view(q.shape[:2]) if lengths is not None else None
    return (scores, lengths) if return_lengths else scores


def select_topk(scores: torch.Tensor, topk: int, *,
                lengths: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Positions of the ``topk`` largest scores of each row, as ``cmp_sparse_indices``.

    scores:   float32 [T, N] / [B, S, N], CUDA; rows may be strided.
    lengths:  int32, one per row: only the first ``lengths`` scores count (default: all).

    Returns int32 [T, 1, topk] / [B, S, 1, topk]: ascending positions, -1 behind them.
    Equal scores go to the lower position.  -inf is never selected; NaN ranks above +inf.
    """
    dev = scores.device
    if dev.type != "cuda":
        raise RuntimeError(f"select_topk runs on a CUDA (sm_100a) device only; got {dev}")
    shape, topk = scores.shape, int(topk)
    if scores.dtype is not torch.float32 or len(shape) not in (2, 3):
        raise ValueError("scores must be float32 [T, N] or [B, S, N]")
    if not 1 <= topk <= _lib.SAS_MAX_TOPK:
        raise ValueError(f"topk must be in [1, 2^30] (got {topk})")
    N = shape[-1]
    rows = shape[0] if len(shape) == 2 else shape[0] * shape[1]
    if rows > _lib.INT32_MAX // 8 or N > _lib.INT32_MAX - 65536:
        raise ValueError(f"scores hold too many rows or columns ({rows} x {N})")
    out = scores.new_empty((*shape[:-1], 1, topk), dtype=torch.int32)
    if lengths is not None:
        if lengths.numel() != rows:
            raise ValueError("lengths must have one entry per row of scores")
        lengths = _lib.dev_i32(lengths, dev)
    if rows == 0:
        return out
    x = scores if len(shape) == 2 else scores.reshape(rows, N)
    row_stride, col_stride = x.stride()
    if (N > 1 and col_stride != 1) or (rows > 1 and row_stride < N):
        x = x.contiguous()
        row_stride = N
    with _lib.on_device(dev) as stream:
        _lib.check("sas_topk_select", _lib.lib().sas_topk_select(
            x.data_ptr(), max(row_stride, N), lengths.data_ptr() if lengths is not None else None,
            rows, N, topk, out.data_ptr(), stream))
    return out


def select_keys(q: torch.Tensor, weights: torch.Tensor, *, key_pool: torch.Tensor,
                block_table: torch.Tensor, cu_seqlens_q: Optional[torch.Tensor] = None,
                seqused_kv: torch.Tensor, topk: int, cmp_ratio: int = 1, layout_q: str = "TND",
                max_keys: Optional[int] = None) -> torch.Tensor:
    """``select_topk(index_scores(...))`` without the whole score matrix: the
    ``cmp_sparse_indices`` ([T, 1, topk] / [B, S, 1, topk] int32) of each token.

    The arguments are ``index_scores``'s; the scores of a part of the tokens at a time are
    held in a workspace of at most 256 MiB (or one token's).
    """
    p, N, keep = _index_params(q, weights, key_pool, block_table, cu_seqlens_q, seqused_kv,
                               cmp_ratio, layout_q, max_keys)
    topk = int(topk)
    if not 1 <= topk <= _lib.SAS_MAX_TOPK:
        raise ValueError(f"topk must be in [1, 2^30] (got {topk})")
    dev, total = q.device, p.total_tokens
    out = torch.empty((*q.shape[:-2], 1, topk), dtype=torch.int32, device=dev)
    if total == 0:
        return out
    stride = max(4, (N + 3) // 4 * 4)
    part = max(1, min(total, _SCORE_WORKSPACE // (4 * stride)))
    scores = torch.empty(part * stride, dtype=torch.float32, device=dev)
    lengths = torch.empty(part, dtype=torch.int32, device=dev)
    err = torch.zeros(4, dtype=torch.int32, device=dev) if _check_device_errors() else None
    p.scores, p.score_stride, p.lengths, p.fill = scores.data_ptr(), stride, lengths.data_ptr(), 0
    p.err = err.data_ptr() if err is not None else None
    L = _lib.lib()
    with _lib.on_device(dev) as stream:
        for t in range(0, total, part):
            p.first_token, p.num_tokens = t, min(part, total - t)
            _lib.check("sas_index_scores", L.sas_index_scores(p, stream))
            _lib.check("sas_topk_select", L.sas_topk_select(
                scores.data_ptr(), stride, lengths.data_ptr(), p.num_tokens, N, topk,
                out.data_ptr() + 4 * t * topk, stream))
    if err is not None:
        _raise_device_error(err)
    del keep
    return out
