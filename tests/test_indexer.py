"""Selection of key positions (``indexer``): index scores against the formula in 64 bits, the
top-k selection exactly, both together, and the whole run from projections to the attention."""

import ctypes as C

import numpy as np
import pytest
import torch

from oracle import sas_oracle as O
from sparse_attn_sharedkv_b200 import _lib, indexer

NEG = float("-inf")


# ---- plain forms ----

def thresholds(cu, kv, ratio):
    """(batch, len) of each token, golden.py:48-62."""
    out = []
    for b in range(len(kv)):
        n = cu[b + 1] - cu[b]
        out += [(b, max(0, (kv[b] - n + s + 1) // ratio)) for s in range(n)]
    return out


def scores_reference(q, w, pool, table, tokens, N):
    """Scores in 64 bits [T, N], and the sums of the magnitudes of what each one adds up."""
    q, w, pool = q.double().cpu(), w.double().cpu(), pool.double().cpu()
    T, H, D = q.shape
    bs = pool.shape[1]
    flat = pool.reshape(-1, D)
    out = torch.full((T, N), NEG, dtype=torch.float64)
    mag = torch.zeros(T, N, dtype=torch.float64)
    for t, (b, n) in enumerate(tokens):
        n = min(n, N)
        j = torch.arange(n)
        lb = j // bs
        blk = torch.full((n,), -1, dtype=torch.long)
        inside = lb < table.shape[1]
        blk[inside] = table[b].long()[lb[inside]]
        ok = (blk >= 0) & (blk < pool.shape[0])
        k = flat[torch.where(ok, blk * bs + j % bs, 0)]
        s = torch.relu(q[t] @ k.T)
        out[t, :n] = torch.where(ok, (w[t, :, None] * s).sum(0), NEG)
        mag[t, :n] = (w[t, :, None].abs() * (q[t].abs() @ k.abs().T)).sum(0)
    return out, mag


def check_scores(got, want, mag, H, D):
    # Products of 16-bit values are exact in fp32.  Each of the D additions of a dot and of the
    # H of the weighted sum, and the product with the weight, is off by at most a whole step
    # (2^-23: the tensor core may cut instead of rounding) of the magnitudes added up.
    got = got.double().cpu()
    assert torch.equal(got == NEG, want == NEG)
    fine = want != NEG
    off = (got[fine] - want[fine]).abs()
    tol = (D + H + 2) * 2.0 ** -23 * mag[fine] + 1e-30
    assert torch.all(off <= tol), float((off / tol).max())


def topk_reference(x, K, lengths=None):
    """Rows of x: NaN first, -0 equal to +0, ties to the lower position, -inf never."""
    x = np.asarray(x, np.float64)
    out = np.full((x.shape[0], K), -1, np.int32)
    for r, row in enumerate(x):
        n = len(row) if lengths is None else max(0, min(len(row), int(lengths[r])))
        v = row[:n]
        v = np.where(np.isnan(v), np.inf, np.where(v == np.inf, np.finfo(np.float64).max, v))
        order = np.argsort(-v, kind="stable")
        best = np.sort(order[v[order] > -np.inf][:K])
        out[r, :len(best)] = best
    return out


# ---- without a GPU ----

def test_topk_reference_orders_special_values():
    x = [[0.0, -0.0, np.nan, np.inf, -np.inf, 1.0, -1.0, 1.0]]
    assert topk_reference(x, 3).tolist() == [[2, 3, 5]]
    assert topk_reference(x, 5).tolist() == [[0, 2, 3, 5, 7]]
    assert topk_reference(x, 9).tolist() == [[0, 1, 2, 3, 5, 6, 7, -1, -1]]
    assert topk_reference(x, 2, [0]).tolist() == [[-1, -1]]


def test_entry_points_refuse_without_a_launch():
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    w = torch.zeros(2, 4)
    kw = dict(key_pool=torch.zeros(1, 4, 1, 64, dtype=torch.bfloat16),
              block_table=torch.zeros(1, 1, dtype=torch.int32),
              cu_seqlens_q=torch.tensor([0, 2]), seqused_kv=torch.tensor([4]))
    with pytest.raises(RuntimeError, match="CUDA"):
        indexer.index_scores(q, w, **kw)
    with pytest.raises(RuntimeError, match="CUDA"):
        indexer.select_keys(q, w, topk=4, **kw)
    with pytest.raises(RuntimeError, match="CUDA"):
        indexer.select_topk(torch.zeros(2, 4), 2)
    L = _lib.lib()
    good = dict(q=16, weights=16, key_pool=16, block_table=16, cu_seqlens_q=16, kv_len=16,
                scores=16, batch=1, total_tokens=4, num_heads=4, head_dim=64, block_size=4,
                num_blocks=1, table_len=1, cmp_ratio=1, num_keys=4, num_tokens=4, score_stride=4)

    def call(**change):
        p = _lib.SasIndexParams(**{**good, **change})
        return L.sas_index_scores(C.byref(p), None)

    assert call(num_tokens=0) == 0
    for bad in (dict(q=None), dict(q=24), dict(key_pool=8), dict(weights=None),
                dict(cu_seqlens_q=None), dict(kv_len=None), dict(scores=None), dict(batch=0),
                dict(cmp_ratio=0), dict(score_stride=3), dict(first_token=1), dict(num_tokens=-1),
                dict(first_token=-1, num_tokens=2), dict(block_size=0), dict(max_q_len=3),
                dict(num_keys=-1)):
        assert call(**bad) == 1, bad
    for bad in (dict(dtype=2), dict(num_heads=129), dict(num_heads=0), dict(head_dim=136),
                dict(head_dim=12), dict(num_blocks=2 ** 30, block_size=2)):
        assert call(**bad) == 2, bad
    assert L.sas_index_scores(None, None) == 1

    def topk(scores=16, stride=8, rows=1, n=8, k=4, out=16):
        return L.sas_topk_select(scores, stride, None, rows, n, k, out, None)

    assert topk(rows=0) == 0
    for bad in (dict(scores=None), dict(out=None), dict(stride=7), dict(rows=-1), dict(n=-1),
                dict(k=0)):
        assert topk(**bad) == 1, bad


def test_topk_entry_refuses_sizes_past_32_bits():
    L = _lib.lib()
    for rows, n, k in ((1, 8, 2 ** 30 + 1), (2 ** 28, 8, 4), (1, 2 ** 31 - 1, 4)):
        assert L.sas_topk_select(16, n, None, rows, n, k, 16, None) == 2, (rows, n, k)


# ---- on a GPU: scores ----

def score_case(seed, q_lens, kv, H, D, bs, ratio=1, dtype=torch.bfloat16, cols=None, spare=3):
    g = torch.Generator().manual_seed(seed)
    B, T = len(q_lens), sum(q_lens)
    N = max(1, max(kv) // ratio) if cols is None else cols
    per = -(-max(1, max(kv) // ratio) // bs)
    q = torch.randn(T, H, D, generator=g).to(dtype)
    w = torch.randn(T, H, generator=g) * (H * D) ** -0.5
    pool = torch.randn(B * per + spare, bs, 1, D, generator=g).to(dtype)
    table = torch.randperm(B * per + spare, generator=g)[:B * per].to(torch.int32).view(B, per)
    cu = [sum(q_lens[:b]) for b in range(B + 1)]
    return q, w, pool, table, cu, list(kv), ratio, N


def run_scores(case, **kw):
    q, w, pool, table, cu, kv, ratio, N = case
    return indexer.index_scores(
        q.cuda(), w.cuda(), key_pool=pool.cuda(), block_table=table.cuda(),
        cu_seqlens_q=torch.tensor(cu, dtype=torch.int32).cuda(),
        seqused_kv=torch.tensor(kv, dtype=torch.int32).cuda(), cmp_ratio=ratio,
        **{"max_keys": N, **kw})


SCORES = [  # q_lens, kv, H, D, block size, ratio
    ((1,), (1,), 1, 8, 1, 1),
    ((1, 1), (700, 513), 64, 128, 64, 1),
    ((1, 1, 1), (4096, 129, 128), 16, 64, 64, 1),
    ((5, 1, 2), (300, 77, 900), 64, 128, 16, 1),
    ((130,), (130,), 64, 128, 64, 1),
    ((33, 0, 9), (600, 50, 9), 24, 96, 5, 1),
    ((7, 20), (515, 20), 128, 128, 128, 1),
    ((3, 3), (1000, 2000), 100, 40, 48, 1),
    ((40, 17), (1031, 2050), 32, 32, 3, 4),
    ((11, 2), (5000, 9000), 8, 128, 32, 128),
    ((6,), (4,), 4, 64, 64, 1),              # fewer keys than tokens: rows that see none
    ((2, 2), (3, 1000), 64, 128, 8, 4),      # rows that see none beside ordinary ones
    ((1,) * 70, tuple(range(1, 700, 10)), 64, 64, 64, 1),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("q_lens, kv, H, D, bs, ratio", SCORES)
def test_gpu_index_scores(q_lens, kv, H, D, bs, ratio, dtype):
    case = score_case(7, q_lens, kv, H, D, bs, ratio, dtype)
    q, w, pool, table, cu, _, _, N = case
    tokens = thresholds(cu, kv, ratio)
    want, mag = scores_reference(q, w, pool, table, tokens, N)
    got, lens = run_scores(case, return_lengths=True)
    check_scores(got, want, mag, H, D)
    assert lens.tolist() == [min(n, N) for _, n in tokens]
    assert torch.equal(run_scores(case), got)  # the same bits again


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [1, 63, 300, 1111])
def test_gpu_index_scores_columns(cols):
    # Fewer columns than keys, and more than the table's pages hold.
    case = score_case(8, (3, 1), (700, 90), 64, 128, 64, cols=cols)
    q, w, pool, table, cu, kv, _, _ = case
    want, mag = scores_reference(q, w, pool, table, thresholds(cu, kv, 1), cols)
    got, lens = run_scores(case, return_lengths=True)
    assert got.shape == (4, cols)
    check_scores(got, want, mag, 64, 128)
    assert lens.tolist() == [min(n, cols) for n in (698, 699, 700, 90)]
    whole = run_scores(case, max_keys=None)
    assert whole.shape == (4, table.shape[1] * 64)
    n = min(cols, whole.shape[1])
    assert torch.equal(whole[:, :n], got[:, :n])


@pytest.mark.gpu
@pytest.mark.parametrize("bs", [5, 64])
def test_gpu_index_scores_bad_pages(bs, monkeypatch):
    case = score_case(9, (4, 1), (333, 200), 24, 64, bs)
    q, w, pool, table, cu, kv, _, N = case
    table[0, 1] = -1
    table[0, 3] = -7
    table[1, 0] = -1
    want, mag = scores_reference(q, w, pool, table, thresholds(cu, kv, 1), N)
    monkeypatch.setenv("SAS_CHECK_DEVICE_ERRORS", "1")
    check_scores(run_scores(case), want, mag, 24, 64)
    table[1, 1] = pool.shape[0]  # past the pool: read as unmapped, and reported
    want, mag = scores_reference(q, w, pool, table, thresholds(cu, kv, 1), N)
    with pytest.raises(RuntimeError, match="site=53"):
        run_scores(case)
    monkeypatch.delenv("SAS_CHECK_DEVICE_ERRORS")
    check_scores(run_scores(case), want, mag, 24, 64)


@pytest.mark.gpu
def test_gpu_index_scores_special_values():
    # Keys that no token sees may hold anything; a NaN in a seen one reaches its score alone.
    case = score_case(10, (3,), (200,), 16, 64, 64)
    q, w, pool, table, cu, kv, _, N = case
    clean = run_scores(case)
    flat = pool.view(-1, 64)
    row = lambda j: int(table[0, j // 64]) * 64 + j % 64
    flat[row(199)] = float("nan")  # the last token alone sees position 199
    for j in range(200, 256):
        flat[row(j)] = float("inf") if j % 2 else float("nan")
    got = run_scores(case)
    assert torch.equal(got[:2], clean[:2]) and torch.equal(got[2, :199], clean[2, :199])
    assert got[2, 199].isnan()
    flat[row(5)] = 3e38
    w.abs_()
    got = run_scores(case)
    assert not (got[:, 5] < 1e38).any() and got[:, :5].isfinite().all()


@pytest.mark.gpu
@pytest.mark.parametrize("H", [12, 16, 20, 33, 64, 100, 128])
def test_gpu_index_scores_infinite_key(H):
    # An infinity in a seen key is that score's, also where the heads do not fill a tile.
    g = torch.Generator().manual_seed(H)
    q = torch.rand(1, H, 64, generator=g).to(torch.bfloat16) + 0.5
    w = torch.rand(1, H, generator=g) + 0.5
    pool = torch.rand(4, 64, 1, 64, generator=g).to(torch.bfloat16)
    pool[1, 3] = float("inf")
    s = run_scores((q, w, pool, torch.tensor([[2, 1, 0]], dtype=torch.int32), [0, 1], [150], 1,
                    150))
    assert s[0, 67] == float("inf") and s[0, :67].isfinite().all() and s[0, 68:].isfinite().all()


@pytest.mark.gpu
@pytest.mark.parametrize("H", [1, 12, 16, 20, 33, 63, 64, 100, 127])
def test_gpu_index_scores_nan_in_the_last_head(H):
    g = torch.Generator().manual_seed(H)
    q = torch.randn(2, H, 64, generator=g).to(torch.bfloat16)
    w = torch.randn(2, H, generator=g)
    pool = torch.randn(4, 64, 1, 64, generator=g).to(torch.bfloat16)
    case = (q, w, pool, torch.tensor([[2, 1, 0]], dtype=torch.int32), [0, 2], [150], 1, 150)
    clean = run_scores(case)
    q[0, H - 1, 5] = float("nan")
    s = run_scores(case)
    assert s[0, :149].isnan().all() and s[0, 149] == NEG and torch.equal(s[1], clean[1])


@pytest.mark.gpu
@pytest.mark.parametrize("H, D, bs", [(16, 128, 64), (64, 128, 64), (128, 64, 48), (40, 128, 20)])
def test_gpu_index_scores_long_runs(H, D, bs):
    # Rows of 131072 keys, so that each pair of CTAs goes through its buffers many times, and
    # groups of few and of many tokens in turn.
    g = torch.Generator().manual_seed(H + bs)
    B, N, per = 41, 131072, 2 * max(1, 128 // H)
    q_len = torch.randint(1, per + 1, (B,), generator=g).tolist()
    q_len[3:7] = [0, 1, 2 * per + 1, per]
    kv = torch.randint(N // 2, N + 1, (B,), generator=g).tolist()
    kv[5], kv[9], kv[11] = N, 77, 0
    cu = [0] + torch.tensor(q_len).cumsum(0).tolist()
    T, blocks, rows = cu[-1], 300, -(-N // bs)
    q = torch.randn(T, H, D, generator=g).to(torch.bfloat16).cuda()
    w = torch.randn(T, H, generator=g).cuda()
    pool = torch.randn(blocks, bs, 1, D, generator=g).to(torch.bfloat16).cuda()
    table = torch.randint(0, blocks, (B, rows), generator=g, dtype=torch.int32)
    table[torch.rand(B, rows, generator=g) < 0.01] = -1
    table = table.cuda()
    i32 = lambda v: torch.tensor(v, dtype=torch.int32).cuda()
    got = indexer.index_scores(q, w, key_pool=pool, block_table=table, cu_seqlens_q=i32(cu),
                               seqused_kv=i32(kv), max_keys=N)
    j = torch.arange(N, device="cuda")
    flat = pool.view(-1, D).double()
    for b in range(B):
        blk = table[b].long()[j // bs]
        k = flat[blk.clamp(min=0) * bs + j % bs]
        for s in range(q_len[b]):
            t = cu[b] + s
            none = (j >= kv[b] - q_len[b] + s + 1) | (blk < 0)
            x = q[t].double()
            want = w[t].double() @ torch.relu(x @ k.T)
            mag = w[t].double().abs() @ (x.abs() @ k.abs().T)
            assert torch.equal(got[t] == NEG, none), (b, s)
            off = torch.where(none, 0.0, (got[t].double() - want).abs())
            tol = (D + H + 2) * 2.0 ** -23 * mag + 1e-30  # as check_scores derives it
            assert torch.all(off <= tol), (b, s, float((off / tol).max()))


@pytest.mark.gpu
def test_gpu_index_scores_bsnd_and_rows_of_no_sequence():
    case = score_case(11, (4, 4, 4), (300, 4, 150), 16, 64, 16)
    q, w, pool, table, cu, kv, _, N = case
    tnd, lens = run_scores(case, return_lengths=True)
    kw = dict(key_pool=pool.cuda(), block_table=table.cuda(), max_keys=N,
              seqused_kv=torch.tensor(kv, dtype=torch.int32).cuda(), return_lengths=True)
    b, bl = indexer.index_scores(q.view(3, 4, 16, 64).cuda(), w.view(3, 4, 16).cuda(),
                                 layout_q="BSND", **kw)
    assert b.shape == (3, 4, N) and torch.equal(b.reshape(12, N), tnd)
    assert torch.equal(bl.view(-1), lens)
    # Ragged BSND: q_len 2, 4, 1; the padded tokens see nothing.
    cu_r = torch.tensor([0, 2, 6, 7], dtype=torch.int32).cuda()
    b, bl = indexer.index_scores(q.view(3, 4, 16, 64).cuda(), w.view(3, 4, 16).cuda(),
                                 layout_q="BSND", cu_seqlens_q=cu_r, **kw)
    assert bl.tolist() == [[299, 300, 0, 0], [1, 2, 3, 4], [150, 0, 0, 0]]
    assert torch.equal(b[0, 2:], torch.full_like(b[0, 2:], NEG))
    assert torch.equal(b[2, 1:], torch.full_like(b[2, 1:], NEG))
    assert torch.equal(b[0, 0, :297], tnd[0, :297]) and torch.equal(b[0, 1, :298], tnd[1, :298])
    # TND tokens behind the last sequence.
    kw["cu_seqlens_q"] = torch.tensor([0, 4, 8, 10], dtype=torch.int32).cuda()
    t, tl = indexer.index_scores(q.cuda(), w.cuda(), **kw)
    assert tl[10:].tolist() == [0, 0] and bool((t[10:] == NEG).all())
    assert torch.equal(t[:8], tnd[:8])


@pytest.mark.gpu
def test_gpu_index_scores_graph_and_new_lengths():
    case = score_case(12, (2, 3), (500, 700), 64, 128, 64)
    q, w, pool, table, cu, kv, _, N = case
    cu_d = torch.tensor(cu, dtype=torch.int32).cuda()
    kv_d = torch.tensor(kv, dtype=torch.int32).cuda()
    args = (q.cuda(), w.cuda())
    kw = dict(key_pool=pool.cuda(), block_table=table.cuda(), cu_seqlens_q=cu_d, seqused_kv=kv_d,
              max_keys=N)
    indexer.index_scores(*args, **kw)
    indexer.select_keys(*args, topk=64, **kw)
    torch.cuda.synchronize()
    first, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(first):
        s = indexer.index_scores(*args, **kw)
    with torch.cuda.graph(second):
        i = indexer.select_keys(*args, topk=64, **kw)
    for lens in ((500, 700), (40, 3), (333, 64)):
        kv_d.copy_(torch.tensor(lens, dtype=torch.int32))
        first.replay()
        second.replay()
        assert torch.equal(s, indexer.index_scores(*args, **kw))
        assert torch.equal(i, indexer.select_keys(*args, topk=64, **kw))
        want, mag = scores_reference(q, w, pool, table, thresholds(cu, lens, 1), N)
        check_scores(s, want, mag, 64, 128)


@pytest.mark.gpu
def test_gpu_refusals():
    case = score_case(13, (2,), (50,), 4, 64, 16)
    q, w, pool, table, cu, kv, _, N = case
    good = dict(q=q.cuda(), weights=w.cuda(), key_pool=pool.cuda(), block_table=table.cuda(),
                cu_seqlens_q=torch.tensor(cu).cuda(), seqused_kv=torch.tensor(kv).cuda())
    indexer.index_scores(**good)
    for change, word in (
            (dict(weights=w.cuda().double()), "weights"), (dict(weights=w.cuda()[:1]), "weights"),
            (dict(weights=w), "weights"), (dict(q=q.cuda().half()), "share"),
            (dict(q=q.cuda().float()), "dtype"), (dict(q=q.cuda()[:, :, :60]), "multiple of 8"),
            (dict(key_pool=pool.cuda()[..., :32]), "share"),
            (dict(cu_seqlens_q=None), "cu_seqlens_q"), (dict(layout_q="BSH"), "layout_q"),
            (dict(layout_q="BSND"), "BSND"), (dict(block_table=table.cuda()[0]), "block_table"),
            (dict(block_table=table.cuda()[:0]), "block_table"),
            (dict(seqused_kv=torch.zeros(0).cuda()), "seqused_kv"), (dict(cmp_ratio=0), "ratio"),
            (dict(max_keys=-1), "max_keys"),
            (dict(q=torch.zeros(2, 129, 64, dtype=torch.bfloat16).cuda(),
                  weights=torch.zeros(2, 129).cuda()), "heads")):
        with pytest.raises(ValueError, match=word):
            indexer.index_scores(**{**good, **change})
    x = torch.zeros(3, 8).cuda()
    for args, word in (((x, 0), "topk"), ((x.half(), 2), "float32"), ((x[0], 2), "float32")):
        with pytest.raises(ValueError, match=word):
            indexer.select_topk(*args)
    with pytest.raises(ValueError, match="lengths"):
        indexer.select_topk(x, 2, lengths=torch.zeros(2))
    with pytest.raises(ValueError, match="topk"):
        indexer.select_keys(topk=0, **good)
    assert indexer.select_topk(x[:0], 2).shape == (0, 1, 2)
    assert indexer.select_topk(x[:, :0], 2).tolist() == [[[-1, -1]]] * 3
    empty = {**good, "q": good["q"][:0], "weights": good["weights"][:0],
             "cu_seqlens_q": torch.tensor([0, 0]).cuda()}
    assert indexer.index_scores(**empty).shape[0] == 0
    assert indexer.select_keys(topk=3, **empty).shape == (0, 1, 3)


@pytest.mark.gpu
def test_gpu_sizes_at_their_ends(monkeypatch):
    monkeypatch.delenv("SAS_CHECK_DEVICE_ERRORS", raising=False)
    case = score_case(13, (2,), (50,), 4, 64, 16)
    q, w, pool, table, cu, kv, _, N = case
    good = dict(q=q.cuda(), weights=w.cuda(), key_pool=pool.cuda(), block_table=table.cuda(),
                cu_seqlens_q=torch.tensor(cu).cuda(), seqused_kv=torch.tensor(kv).cuda())
    x = torch.zeros(3, 8).cuda()
    for k in (-1, 2 ** 30 + 1, 2 ** 32 + 2):
        with pytest.raises(ValueError, match="topk"):
            indexer.select_topk(x, k)
        with pytest.raises(ValueError, match="topk"):
            indexer.select_keys(topk=k, **good)
    with pytest.raises(ValueError, match="ratio"):
        indexer.index_scores(**{**good, "cmp_ratio": 2 ** 32 + 1})
    # No columns, no pages, no pool.
    s, n = indexer.index_scores(max_keys=0, return_lengths=True, **good)
    assert s.shape == (2, 0) and n.tolist() == [0, 0]
    for change in (dict(block_table=table.cuda()[:, :0]), dict(key_pool=pool.cuda()[:0])):
        s, n = indexer.index_scores(max_keys=9, return_lengths=True, **{**good, **change})
        assert bool((s == NEG).all()) and s.shape == (2, 9) and n.tolist() == [9, 9]
        assert bool((indexer.select_keys(topk=3, max_keys=9, **{**good, **change}) == -1).all())
    # A page of an empty pool is one past it: reported, where that is asked for.
    monkeypatch.setenv("SAS_CHECK_DEVICE_ERRORS", "1")
    with pytest.raises(RuntimeError, match="site=53"):
        indexer.index_scores(**{**good, "key_pool": pool.cuda()[:0]})


# ---- on a GPU: selection ----

def topk_rows(kind, rows, N, g):
    x = torch.randn(rows, N, generator=g)
    if kind == "ties":
        return x.to(torch.bfloat16).float()
    if kind == "equal":
        return torch.full((rows, N), -2.5)
    if kind == "two":  # one of two neighbouring floats
        return torch.where(x > 0.3, 1.0, float(np.nextafter(np.float32(1), np.float32(2))))
    if kind == "wide":  # magnitudes over the whole range of the type, both signs
        return torch.sign(x) * torch.exp(30 * torch.randn(rows, N, generator=g))
    if kind == "close":  # a spread of a few thousand steps of the type
        return 1.0 + (x * 1000).round() * 2.0 ** -23
    if kind == "tiny":  # subnormal values and signed zeros
        return (x * 3).round() * 2.0 ** -149 * torch.where(x > 1, -1.0, 1.0)
    if kind == "outlier":
        x[:, ::97] = 1e30
        x[:, 1::97] = -1e30
        return x
    if kind == "special":
        x[:, ::7] = NEG
        x[:, 3::11] = float("inf")
        x[:, 5::13] = float("nan")
        x[:, 6::17] = -0.0
        x[:, 7::17] = 0.0
        return x
    if kind == "masked":  # almost everything masked by -inf or the type's lowest value
        x[:, torch.rand(N, generator=g) < 0.9] = NEG
        x[:, torch.rand(N, generator=g) < 0.05] = torch.finfo(torch.float32).min
        return x
    if kind == "up":
        return torch.arange(N, dtype=torch.float32).expand(rows, N).contiguous()
    if kind == "down":
        return -torch.arange(N, dtype=torch.float32).expand(rows, N).contiguous()
    return x


KINDS = ("normal", "ties", "equal", "two", "wide", "close", "tiny", "outlier", "special", "masked",
         "up", "down")


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows, N, K", [(1, 1, 1), (3, 5, 9), (2, 100, 100), (5, 513, 64),
                                        (3, 2049, 2048), (4, 4096, 1), (2, 4097, 512),
                                        (3, 9000, 2048), (2, 17001, 700), (60, 16390, 100),
                                        (2, 33000, 2000), (2, 131072, 2048), (1, 140001, 2048),
                                        (300, 700, 130)])
def test_gpu_select_topk(rows, N, K, kind):
    g = torch.Generator().manual_seed(N + K)
    x = topk_rows(kind, rows, N, g)
    lengths = torch.randint(0, N + 1, (rows,), generator=g, dtype=torch.int32)
    d = x.cuda()
    assert np.array_equal(indexer.select_topk(d, K)[:, 0].cpu().numpy(), topk_reference(x, K))
    got = indexer.select_topk(d, K, lengths=lengths.cuda())
    assert got.shape == (rows, 1, K) and got.dtype == torch.int32
    assert np.array_equal(got[:, 0].cpu().numpy(), topk_reference(x, K, lengths))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows, N, K", [(310, 3001, 1500), (300, 6007, 512), (299, 16000, 2048)])
def test_gpu_select_topk_many_rows(rows, N, K, kind):
    # More than two rows for each SM, of which some are empty, shorter than K or whole.
    g = torch.Generator().manual_seed(N + K)
    x = topk_rows(kind, rows, N, g)
    lengths = torch.randint(0, N + 1, (rows,), generator=g, dtype=torch.int32)
    lengths[:6] = torch.tensor([0, N, 1, K, K + 1, N])
    d = x.cuda()
    got = indexer.select_topk(d, K, lengths=lengths.cuda())
    assert np.array_equal(got[:, 0].cpu().numpy(), topk_reference(x, K, lengths))
    assert torch.equal(indexer.select_topk(d, K, lengths=lengths.cuda()), got)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows, N, K", [(3, 200001, 2048), (3, 270001, 700), (2, 600011, 5000),
                                        (1, 1000003, 300000)])
def test_gpu_select_topk_long_rows(rows, N, K, kind):
    g = torch.Generator().manual_seed(N + K)
    x = topk_rows(kind, rows, N, g)
    lengths = torch.randint(0, N + 1, (rows,), generator=g, dtype=torch.int32)
    d = x.cuda()
    assert np.array_equal(indexer.select_topk(d, K)[:, 0].cpu().numpy(), topk_reference(x, K))
    got = indexer.select_topk(d, K, lengths=lengths.cuda())
    assert np.array_equal(got[:, 0].cpu().numpy(), topk_reference(x, K, lengths))


@pytest.mark.gpu
def test_gpu_select_topk_strides_lengths_and_stream():
    g = torch.Generator().manual_seed(3)
    x = torch.randn(6, 1003, generator=g)
    d = x.cuda()
    want = topk_reference(x[:, 1:1000], 77)
    assert np.array_equal(indexer.select_topk(d[:, 1:1000], 77)[:, 0].cpu().numpy(), want)
    assert np.array_equal(indexer.select_topk(d[:, 1:1000].t().contiguous().t(), 77)[:, 0]
                          .cpu().numpy(), want)
    assert np.array_equal(indexer.select_topk(d[:1].expand(3, 1003), 5)[:, 0].cpu().numpy(),
                          topk_reference(x[:1].expand(3, 1003), 5))
    odd = torch.tensor([-3, 0, 1, 5000, 1003, 2])
    assert np.array_equal(indexer.select_topk(d, 7, lengths=odd.cuda())[:, 0].cpu().numpy(),
                          topk_reference(x, 7, odd))
    b = indexer.select_topk(d.view(2, 3, 1003), 9, lengths=odd.view(2, 3).cuda())
    assert b.shape == (2, 3, 1, 9)
    assert torch.equal(b.view(6, 1, 9), indexer.select_topk(d, 9, lengths=odd.cuda()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        s = indexer.select_topk(d, 9, lengths=odd.cuda())
    side.synchronize()
    assert torch.equal(s, b.view(6, 1, 9))
    graph = torch.cuda.CUDAGraph()
    lens = odd.to(torch.int32).cuda()
    with torch.cuda.graph(graph):
        s = indexer.select_topk(d, 9, lengths=lens)
    d.copy_(d.flip(1))
    lens.fill_(500)
    graph.replay()
    assert np.array_equal(s[:, 0].cpu().numpy(), topk_reference(x.flip(1), 9, [500] * 6))


@pytest.mark.gpu
@pytest.mark.parametrize("work", [1, 40_000, 64 << 20])
def test_gpu_select_keys_is_scores_then_topk(work, monkeypatch):
    monkeypatch.setattr(indexer, "_SCORE_WORKSPACE", work)
    case = score_case(21, (30, 1, 0, 45), (900, 333, 8, 45), 24, 96, 16, 1)
    q, w, pool, table, cu, kv, ratio, N = case
    args = (q.cuda(), w.cuda())
    kw = dict(key_pool=pool.cuda(), block_table=table.cuda(), max_keys=N,
              cu_seqlens_q=torch.tensor(cu, dtype=torch.int32).cuda(),
              seqused_kv=torch.tensor(kv, dtype=torch.int32).cuda())
    got = indexer.select_keys(*args, topk=100, **kw)
    s, lens = indexer.index_scores(*args, return_lengths=True, **kw)
    assert torch.equal(got, indexer.select_topk(s, 100, lengths=lens))
    assert torch.equal(got, indexer.select_topk(s, 100))
    kw.pop("cu_seqlens_q")
    b = indexer.select_keys(args[0].view(4, 19, 24, 96), args[1].view(4, 19, 24), topk=100,
                            layout_q="BSND", **kw)
    s = indexer.index_scores(args[0].view(4, 19, 24, 96), args[1].view(4, 19, 24),
                             layout_q="BSND", **kw)
    assert b.shape == (4, 19, 1, 100) and torch.equal(b, indexer.select_topk(s, 100))


# ---- the run from projections to the attention ----

@pytest.mark.gpu
@pytest.mark.parametrize("new", [(1, 1, 1), (130, 1, 37)])
def test_gpu_projections_to_attention(new):
    from sparse_attn_sharedkv_b200.api import sparse_attn_sharedkv
    from sparse_attn_sharedkv_b200.kv_cache import append_paged_kv_norm_rope
    from sparse_attn_sharedkv_b200.rope import norm_rope
    g = torch.Generator().manual_seed(5)
    dev, H, D, Hi, Di, K, bs = "cuda", 64, 576, 32, 128, 128, 64
    rnd = lambda *s: (0.5 * torch.randn(*s, generator=g)).to(torch.bfloat16)
    before = [700, 64, 300]
    B, T = len(new), sum(new)
    kv = [n + m for n, m in zip(before, new)]
    per = -(-max(kv) // bs)
    table = torch.randperm(B * per, generator=g).to(torch.int32).view(B, per).to(dev)
    freq = 10000.0 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64)
    ang = torch.arange(2048, dtype=torch.float64)[:, None] * freq
    cos, sin = ang.cos().float().to(dev), ang.sin().float().to(dev)
    w_kv = (1 + 0.1 * torch.randn(512, generator=g)).to(dev)
    pool = torch.zeros(B * per, bs, 1, D, dtype=torch.bfloat16, device=dev)
    ipool = torch.zeros(B * per, bs, 1, Di, dtype=torch.bfloat16, device=dev)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)

    def append(n, start):
        cu = i32([sum(n[:b]) for b in range(B + 1)])
        rows, irows = rnd(sum(n), D).to(dev), rnd(sum(n), Di).to(dev)
        assert append_paged_kv_norm_rope(pool, table, rows, cu, i32(start), cos, sin, norm_dim=512,
                                         norm_weight=w_kv, check_errors=True) is None
        assert append_paged_kv_norm_rope(ipool, table, irows, cu, i32(start), cos, sin,
                                         norm_dim=Di, interleaved=False,
                                         check_errors=True) is None
        return cu

    append(before, [0] * B)
    cu = append(list(new), before)
    positions = torch.cat([torch.arange(n, n + m) for n, m in zip(before, new)]).to(dev)
    q = norm_rope(rnd(T, H, D).to(dev), positions, cos, sin, norm_dim=512)
    qi = norm_rope(rnd(T, Hi, Di).to(dev), positions, cos, sin, interleaved=False)
    wi = torch.randn(T, Hi, generator=g).to(dev)
    kw = dict(block_table=table, cu_seqlens_q=cu, seqused_kv=i32(kv), max_keys=max(kv))
    idx = indexer.select_keys(qi, wi, key_pool=ipool, topk=K, **kw)
    # Every selected position scores at least what the best one left out does, as far as fp32
    # tells them apart.
    tokens = thresholds(cu.tolist(), kv, 1)
    want, mag = scores_reference(qi, wi, ipool, table.cpu(), tokens, max(kv))
    for t, (b, n) in enumerate(tokens):
        got = idx[t, 0].cpu()
        got = got[got >= 0].long()
        assert len(got) == min(n, K) and torch.equal(got, got.unique())
        left = torch.ones(n, dtype=torch.bool)
        left[got] = False
        if left.any():
            slack = 2 * (Di + Hi + 2) * 2.0 ** -23 * float(mag[t].max())
            assert float(want[t, got].min()) >= float(want[t, :n][left].max()) - slack
    call = dict(ori_kv=pool, ori_block_table=table, cmp_kv=pool, cmp_block_table=table,
                cmp_sparse_indices=idx, cu_seqlens_q=cu, seqused_kv=i32(kv),
                sinks=torch.full((H,), NEG, device=dev), softmax_scale=D ** -0.5, cmp_ratio=1,
                ori_win_left=-1)
    out, lse = sparse_attn_sharedkv(q, return_softmax_lse=True, **call)
    f = lambda t: t.to(torch.float32).cpu().numpy()
    i = lambda t: t.to(torch.int64).cpu().numpy()
    ref, ref_lse = O.forward(
        q=f(q), ori_kv=f(pool), ori_block_table=i(table), seqused_kv=kv, sinks=f(call["sinks"]),
        softmax_scale=D ** -0.5, layout_q="TND", cu_seqlens_q=i(cu).tolist(), cmp_kv=f(pool),
        cmp_block_table=i(table), cmp_sparse_indices=i(idx), cmp_ratio=1, ori_win_left=-1,
        head_dim_v=512, dtype="bf16")
    assert np.abs(f(out) - ref).max() <= 2e-2 and np.abs(f(lse) - ref_lse).max() <= 2e-4
    # The same step captured (with the plan built on the device) and replayed.
    graph = torch.cuda.CUDAGraph()
    sparse_attn_sharedkv(q, device_plan=True, **call)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        again = indexer.select_keys(qi, wi, key_pool=ipool, topk=K, **kw)
        o2 = sparse_attn_sharedkv(q, device_plan=True, **{**call, "cmp_sparse_indices": again})
    graph.replay()
    assert torch.equal(again, idx) and torch.equal(o2, out)
