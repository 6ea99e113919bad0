"""What ``include/sas.h`` says of ``sas_index_scores`` beyond the scores themselves."""

import numpy as np
import pytest
import torch

from sparse_attn_sharedkv_b200 import _lib, indexer

from .test_indexer import NEG, check_scores, score_case, scores_reference, thresholds, \
    topk_reference


def i32(v):
    return torch.tensor(v, dtype=torch.int32).cuda()


def raw_scores(q, w, pool, table, cu, kv, cols, stride=None, scores=None, lengths=None, **change):
    """``sas_index_scores`` of CUDA tensors, its outputs where the caller has them."""
    T, H, D = q.shape
    p = _lib.SasIndexParams(
        q=q.data_ptr(), weights=w.data_ptr(), key_pool=pool.data_ptr(),
        block_table=table.data_ptr(), cu_seqlens_q=cu.data_ptr(), kv_len=kv.data_ptr(),
        scores=scores.data_ptr(), lengths=lengths.data_ptr() if lengths is not None else None,
        batch=kv.numel(), total_tokens=T, num_heads=H, head_dim=D,
        dtype=_lib.DTYPE_BF16 if q.dtype == torch.bfloat16 else _lib.DTYPE_FP16,
        block_size=pool.shape[1], num_blocks=pool.shape[0], table_len=table.shape[1],
        cmp_ratio=1, num_keys=cols, num_tokens=T, fill=1, score_stride=stride or cols)
    for name, value in change.items():
        setattr(p, name, value)
    _lib.check("sas_index_scores", _lib.lib().sas_index_scores(
        p, torch.cuda.current_stream().cuda_stream))


@pytest.mark.gpu
@pytest.mark.parametrize("H", [8, 64, 128])
@pytest.mark.parametrize("before, behind", [(1, 0), (3, 2), (17, 1), (400, 0)])
def test_gpu_tokens_of_no_sequence(H, before, behind):
    q_lens, kv = (5, 0, 9), (700, 30, 90)
    q, w, pool, table, cu, _, _, N = score_case(31, q_lens, kv, H, 64, 16)
    want, mag = scores_reference(q, w, pool, table, thresholds(cu, kv, 1), N)
    lens = [0] * before + [n for _, n in thresholds(cu, kv, 1)] + [0] * behind
    pad = lambda t: torch.cat([t[:1].expand(before, *t.shape[1:]), t,
                               t[:1].expand(behind, *t.shape[1:])]).contiguous().cuda()
    qp, wp, cup = pad(q), pad(w), i32([before + c for c in cu])
    T = qp.shape[0]
    # Outputs that held something else, so that a row left out shows.
    scores = torch.full((T, N), 123.0, device="cuda")
    lengths = torch.full((T,), 77, dtype=torch.int32, device="cuda")
    raw_scores(qp, wp, pool.cuda(), table.cuda(), cup, i32(kv), N, scores=scores, lengths=lengths)
    assert lengths.tolist() == lens
    inside = scores[before:T - behind]
    check_scores(inside, want, mag, H, 64)
    assert bool((scores[:before] == NEG).all()) and bool((scores[T - behind:] == NEG).all())
    # Without the fill their rows stay as they were.
    left = torch.full((T, N), 123.0, device="cuda")
    raw_scores(qp, wp, pool.cuda(), table.cuda(), cup, i32(kv), N, scores=left, lengths=lengths,
               fill=0)
    assert lengths.tolist() == lens and bool((left[:before] == 123.0).all())
    assert bool((left[T - behind:] == 123.0).all())
    # A part of the tokens that starts between the ones of no sequence.
    first = before // 2
    part = torch.full((T - first, N), 123.0, device="cuda")
    raw_scores(qp, wp, pool.cuda(), table.cuda(), cup, i32(kv), N, scores=part,
               lengths=lengths[first:], first_token=first, num_tokens=T - first)
    assert torch.equal(part, scores[first:]) and lengths.tolist() == lens
    # The selection of such a batch.
    idx = indexer.select_keys(qp, wp, key_pool=pool.cuda(), block_table=table.cuda(),
                              cu_seqlens_q=cup, seqused_kv=i32(kv), topk=40, max_keys=N)
    assert np.array_equal(idx[:, 0].cpu().numpy(),
                          topk_reference(scores.cpu().numpy(), 40, lens))
    assert bool((idx[:before] == -1).all())


@pytest.mark.gpu
@pytest.mark.parametrize("bs", [5, 64])
@pytest.mark.parametrize("bad", [0, 2, 3])
def test_gpu_page_past_the_pool_names_its_sequence(bs, bad, monkeypatch):
    kv = (333, 7, 200, 900)
    q, w, pool, table, cu, _, _, N = score_case(9, (4, 1, 2, 1), kv, 24, 64, bs)
    page = pool.shape[0] + 5
    table[bad, 1] = page
    table[1, 1] = page + 1  # of a position that its sequence does not have
    if bs == 5:
        table[1, 1:3] = torch.tensor([1, page + 1])
    monkeypatch.setenv("SAS_CHECK_DEVICE_ERRORS", "1")
    kw = dict(key_pool=pool.cuda(), block_table=table.cuda(), cu_seqlens_q=i32(cu),
              seqused_kv=i32(kv), max_keys=N)
    with pytest.raises(RuntimeError, match=f"code=6 site=53 detail={page} {bad}$"):
        indexer.index_scores(q.cuda(), w.cuda(), **kw)
    with pytest.raises(RuntimeError, match=f"code=6 site=53 detail={page} {bad}$"):
        indexer.select_keys(q.cuda(), w.cuda(), topk=8, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("offset, spare", [(1, 0), (0, 1), (3, 6), (0, 0), (0, 4)])
@pytest.mark.parametrize("cols", [257, 1023, 2051])
def test_gpu_scores_of_any_alignment(cols, offset, spare):
    # Rows that start anywhere and follow at any stride, columns several tiles behind the last
    # position that a token sees; what lies between and behind the rows stays.
    q, w, pool, table, cu, kv, _, _ = score_case(33, (9, 1, 4), (40, 700, 4), 24, 64, 16)
    want, mag = scores_reference(q, w, pool, table, thresholds(cu, kv, 1), cols)
    T, stride = q.shape[0], cols + spare
    buf = torch.full((offset + T * stride + 8,), 123.0, device="cuda")
    args = (q.cuda(), w.cuda(), pool.cuda(), table.cuda(), i32(cu), i32(kv), cols)
    raw_scores(*args, stride=stride, scores=buf[offset:])
    rows = buf[offset:offset + T * stride].view(T, stride)
    check_scores(rows[:, :cols], want, mag, 24, 64)
    kw = dict(key_pool=args[2], block_table=args[3], cu_seqlens_q=args[4], seqused_kv=args[5])
    assert torch.equal(rows[:, :cols], indexer.index_scores(*args[:2], max_keys=cols, **kw))
    buf.as_strided((T, cols), (stride, 1), offset).fill_(123.0)
    assert bool((buf == 123.0).all())
