"""Norm and rotation of rows: query heads (``rope.norm_rope``) and key rows on their way into
a paged cache (``kv_cache.append_paged_kv_norm_rope``), against the formula in 64 bits."""

import ctypes as C

import numpy as np
import pytest
import torch

from sparse_attn_sharedkv_b200 import _lib
from sparse_attn_sharedkv_b200.rope import _rows_overlap, row_transform

EPS = 1e-6


def tables(rope, positions=4096, device="cpu"):
    freq = 10000.0 ** (-torch.arange(0, rope, 2, dtype=torch.float64) / rope)
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * freq
    return angle.cos().float().to(device), angle.sin().float().to(device)


def reference(x, pos, cos, sin, norm, weight, interleaved, inverse=False):
    """Rows x [..., D] (pos [...]) in 64 bits, and for each column the magnitude that the fp32
    steps' errors are relative to: the two columns of a rotated pair."""
    y = x.double().cpu().numpy().copy()
    D = y.shape[-1]
    if norm:
        y[..., :norm] /= np.sqrt((y[..., :norm] ** 2).mean(-1, keepdims=True) + EPS)
        if weight is not None:
            y[..., :norm] *= weight.double().cpu().numpy()
    mag = np.abs(y)
    if cos is not None:
        half = cos.shape[1]
        p = pos.cpu().numpy()
        co, si = cos.double().cpu().numpy()[p], sin.double().cpu().numpy()[p]
        if inverse:
            si = -si
        t = y[..., D - 2 * half:]
        first, second = ((slice(0, None, 2), slice(1, None, 2)) if interleaved
                         else (slice(0, half), slice(half, None)))
        a, b = t[..., first].copy(), t[..., second].copy()
        t[..., first], t[..., second] = a * co - b * si, b * co + a * si
        m = mag[..., D - 2 * half:]
        m[..., first] = m[..., second] = np.abs(a) + np.abs(b)
    return y, mag


def check(got, want, mag, dtype):
    # One rounding to 16 bits (half a step of the value; fp16 below 2^-14 has the fixed step
    # 2^-24), and the fp32 steps before it: a square sum over at most 1024 columns whose
    # shuffle tree adds at most 40 in a row (error 20 * 2^-24 of the norm factor), the
    # reciprocal root (2 steps) and five products and sums, each 2^-24: below 32 * 2^-24.
    half_step = torch.finfo(dtype).eps / 2
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    tol = half_step * np.abs(want) + (1 + half_step) * 32 * 2.0 ** -24 * mag + tiny
    off = np.abs(got.double().cpu().numpy() - want)
    assert np.all(off <= tol), float((off / tol).max())


# ---- without a GPU ----

@pytest.mark.parametrize("change, word", [
    (dict(dtype=torch.float32), "bfloat16 or float16"),
    (dict(head_dim=100), "multiple of 8"),
    (dict(head_dim=2048), "multiple of 8"),
    (dict(norm_dim=12), "norm_dim"),
    (dict(norm_dim=640), "norm_dim"),
    (dict(sin=None), "together"),
    (dict(cos=torch.zeros(8, 12), sin=torch.zeros(8, 12)), "rope_dim"),
    (dict(cos=torch.zeros(8, 32, dtype=torch.float64)), "float32"),
    (dict(cos=torch.zeros(9, 32)), "positions"),
    (dict(norm_weight=torch.ones(8)), "norm_weight"),
    (dict(norm_weight=torch.ones(512, dtype=torch.float16)), "norm_weight"),
    (dict(norm_dim=0, norm_weight=None, cos=None, sin=None), "nothing to do"),
    (dict(head_dim=1024, cos=torch.zeros(8, 144), sin=torch.zeros(8, 144)), "rope_dim"),
    (dict(cos=tables(64, 8)[0].view(-1)[2:34].view(1, 32), sin=torch.zeros(1, 32)), "aligned"),
    (dict(eps=-1.0), "eps"),
])
def test_transform_refuses(change, word):
    cos, sin = tables(64, 8)
    kw = dict(dtype=torch.bfloat16, device=torch.device("cpu"), head_dim=576, cos=cos, sin=sin,
              norm_dim=512, norm_weight=torch.ones(512), eps=EPS, interleaved=True, inverse=False)
    row_transform(**kw)
    kw.update(change)
    with pytest.raises(ValueError, match=word):
        row_transform(**kw)


def test_transform_refuses_empty_tables():
    none = torch.zeros(0, 32)
    with pytest.raises(ValueError, match="no position"):
        row_transform(torch.bfloat16, torch.device("cpu"), 576, none, none, 512, None, EPS, True,
                      False)


def test_entry_points_refuse_without_a_launch():
    from sparse_attn_sharedkv_b200.kv_cache import append_paged_kv_norm_rope
    from sparse_attn_sharedkv_b200.rope import norm_rope
    cos, sin = tables(64, 8)
    x = torch.zeros(1, 1, 576, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA"):
        norm_rope(x, torch.zeros(1, dtype=torch.int32), cos, sin)
    with pytest.raises(RuntimeError, match="CUDA"):
        append_paged_kv_norm_rope(x, torch.zeros(1, 1), x[0], torch.zeros(2), torch.zeros(1),
                                  cos, sin)
    # The C entries: a bad transform, stride, alignment or null pointer returns a code.
    L = _lib.lib()
    good = dict(cos=16, sin=16, table_rows=4, head_dim=576, norm_dim=512, rope_dim=64, eps=1e-6)

    def call(x=16, xs=576, out=16, tokens=1, pos=16, tr=None, **change):
        t = _lib.SasRowTransform(**{**good, **change}) if tr is None else tr
        return L.sas_norm_rope(C.byref(t), x, xs, 576, out, 576, 576, tokens, 1, pos, 0, None,
                               None)

    assert call(tokens=0) == 0
    assert call(tokens=-1) == 1
    for bad in (dict(x=24), dict(x=None), dict(out=None), dict(pos=None), dict(xs=580),
                dict(head_dim=20), dict(norm_dim=-8), dict(rope_dim=24), dict(rope_dim=640),
                dict(cos=None), dict(sin=4), dict(eps=float("nan")), dict(norm_weight=4)):
        assert call(**bad) == 1, bad
    for bad in (dict(dtype=2), dict(head_dim=1032), dict(norm_weight=16, weight_dtype=1)):
        assert call(**bad) == 2, bad

    def append(pool=16, total=1, batch=1, bs=64, ratio=1, rows=16):
        t = _lib.SasRowTransform(**good)
        return L.sas_kv_append_norm_rope(C.byref(t), pool, 1, bs, 16, 1, rows, 16, 16, batch,
                                         total, ratio, None, None)

    assert append(total=0) == 0
    for bad in (dict(pool=None), dict(rows=24), dict(batch=0), dict(bs=0), dict(ratio=0),
                dict(total=-1)):
        assert append(**bad) == 1, bad


def test_rows_overlap():
    assert not _rows_overlap((4, 3), (48, 16), 16) and not _rows_overlap((3, 4), (16, 48), 16)
    assert not _rows_overlap((4, 1), (48, 0), 16) and not _rows_overlap((4, 3), (48, 16), 8)
    assert _rows_overlap((4, 3), (0, 16), 16) and _rows_overlap((2, 3), (16, 16), 16)


# ---- on a GPU ----

ROWS = [  # D, rope, norm, weight dtype (None: ones), interleaved
    (576, 64, 512, torch.float32, True),
    (576, 64, 512, torch.float32, False),
    (512, 64, 512, None, True),
    (512, 64, 512, "row", False),
    (576, 64, 0, None, True),
    (576, 0, 576, torch.float32, True),
    (128, 64, 128, torch.float32, False),
    (128, 128, 0, None, False),
    (64, 64, 64, "row", True),
    (64, 16, 8, torch.float32, False),
    (200, 48, 136, torch.float32, False),
    (264, 32, 40, "row", True),
    (1024, 64, 1024, torch.float32, True),
    (8, 0, 8, torch.float32, True),
]


def row_case(D, rope, norm, wt, dtype, n, seed, positions=4096):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, D, generator=g).to(dtype).cuda()
    cos, sin = tables(rope, positions, "cuda") if rope else (None, None)
    w = None
    if wt is not None:
        w = (1 + 0.3 * torch.randn(norm, generator=g)).to(dtype if wt == "row" else wt).cuda()
    pos = torch.randint(0, positions, (n,), generator=g).cuda()
    return x, cos, sin, w, pos


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D, rope, norm, wt, inter", ROWS)
def test_gpu_norm_rope(D, rope, norm, wt, inter, dtype):
    from sparse_attn_sharedkv_b200.rope import norm_rope
    for T, H in ((1, 1), (1, 128), (33, 3), (257, 16)):
        x, cos, sin, w, _ = row_case(D, rope, norm, wt, dtype, T * H, T)
        x = x.view(T, H, D)
        pos = torch.randint(0, 4096, (T,), dtype=torch.int32).cuda()
        kw = dict(norm_dim=norm, norm_weight=w, eps=EPS, interleaved=inter)
        want, mag = reference(x, pos[:, None].expand(T, H), cos, sin, norm, w, inter)
        y = norm_rope(x, pos, cos, sin, **kw)
        check(y, want, mag, dtype)
        assert torch.equal(norm_rope(x, pos.long(), cos, sin, **kw), y)
        z = x.clone()
        assert norm_rope(z, pos, cos, sin, out=z, **kw) is z and torch.equal(z, y)
        if T > 1:
            b = norm_rope(x[:32].view(2, 16, H, D), pos[:32].view(2, 16), cos, sin, **kw)
            assert b.shape == (2, 16, H, D) and torch.equal(b.view(32, H, D), y[:32])
        if rope:
            want, mag = reference(x, pos[:, None].expand(T, H), cos, sin, norm, w, inter, True)
            check(norm_rope(x, pos, cos, sin, inverse=True, **kw), want, mag, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("D, rope, norm, wt, inter", [
    *[ROWS[i] for i in (0, 1, 2, 3, 6, 8, 10, 11)],
    (576, 256, 576, torch.float32, True), (576, 256, 576, "row", False),
    (320, 144, 200, torch.float32, True), (1024, 256, 512, None, False)])
def test_gpu_norm_rope_many_rows_and_wide_rotations(D, rope, norm, wt, inter):
    # 12000 rows: more than all blocks that are resident at once take in one step.
    from sparse_attn_sharedkv_b200.rope import norm_rope
    for T, H in ((300, 40), (3, 5)):
        x, cos, sin, w, _ = row_case(D, rope, norm, wt, torch.bfloat16, T * H, D + rope)
        x = x.view(T, H, D)
        pos = torch.randint(0, 4096, (T,), generator=torch.Generator().manual_seed(T)).cuda()
        kw = dict(norm_dim=norm, norm_weight=w, eps=EPS, interleaved=inter)
        want, mag = reference(x, pos[:, None].expand(T, H), cos, sin, norm, w, inter)
        y = norm_rope(x, pos, cos, sin, **kw)
        check(y, want, mag, torch.bfloat16)
        bad = torch.arange(T, device="cuda") % 7 == 2  # rows outside the tables, between others
        z = x.clone()
        norm_rope(z, torch.where(bad, 4096 - 8191 * (pos % 2), pos), cos, sin, out=z, **kw)
        if rope:
            y[bad] = 0
        assert torch.equal(z, y)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D, rope, norm, wt, inter", [
    *[ROWS[i] for i in (6, 7, 8, 9, 10)], (128, 64, 128, "row", True), (256, 256, 128, None, True),
    (256, 64, 256, torch.float32, False), (64, 64, 0, None, False)])
def test_gpu_norm_rope_many_narrow_rows(D, rope, norm, wt, inter, dtype):
    from sparse_attn_sharedkv_b200.rope import norm_rope
    T, H = 641, 32
    x, cos, sin, w, _ = row_case(D, rope, norm, wt, dtype, T * H, D + rope)
    x = x.view(T, H, D)
    pos = torch.randint(0, 4096, (T,), generator=torch.Generator().manual_seed(T)).cuda()
    kw = dict(norm_dim=norm, norm_weight=w, eps=EPS, interleaved=inter)
    want, mag = reference(x, pos[:, None].expand(T, H), cos, sin, norm, w, inter)
    y = norm_rope(x, pos, cos, sin, **kw)
    check(y, want, mag, dtype)
    norm_rope(x, pos, cos, sin, out=x, **kw)
    assert torch.equal(x, y)


@pytest.mark.gpu
def test_gpu_norm_rope_strided_and_far_apart():
    from sparse_attn_sharedkv_b200.rope import norm_rope
    x, cos, sin, w, _ = row_case(576, 64, 512, torch.float32, torch.bfloat16, 5 * 7 * 2, 3)
    pos = torch.arange(5, dtype=torch.int32).cuda() * 1000
    wide = x.view(5, 7, 2 * 576)
    kw = dict(norm_dim=512, norm_weight=w)
    for part in (wide[..., :576], wide[..., 576:], wide.view(7, 5, 1152)[..., 576:].transpose(0, 1),
                 wide.view(5, 7, 1152)[..., 4:580]):  # the last one is not 16-byte aligned
        y = norm_rope(part, pos, cos, sin, **kw)
        assert torch.equal(y, norm_rope(part.contiguous(), pos, cos, sin, **kw))
    # A view transformed in place leaves what lies between its rows.
    before, part = wide.clone(), wide[..., 576:]
    y = norm_rope(part, pos, cos, sin, **kw)
    norm_rope(part, pos, cos, sin, out=part, **kw)
    assert torch.equal(part, y) and torch.equal(wide[..., :576], before[..., :576])
    # One row of a broadcast input; a broadcast output is refused.
    one = x[:1].view(1, 1, 576).expand(5, 7, 576)
    assert torch.equal(norm_rope(one, pos, cos, sin, **kw),
                       norm_rope(one.contiguous(), pos, cos, sin, **kw))
    with pytest.raises(ValueError, match="overlap"):
        norm_rope(one.contiguous(), pos, cos, sin, out=one, **kw)
    # Element offsets past 32 bits: two tokens 2^31 + 8 elements apart.
    try:
        big = torch.empty(2 ** 31 + 8 + 576, dtype=torch.bfloat16, device="cuda")
    except torch.OutOfMemoryError:
        return
    two = big.as_strided((2, 1, 576), (2 ** 31 + 8, 576, 1))
    two.copy_(x[:2].view(2, 1, 576))
    assert torch.equal(norm_rope(two, pos[:2], cos, sin, **kw),
                       norm_rope(x[:2].view(2, 1, 576), pos[:2], cos, sin, **kw))


@pytest.mark.gpu
def test_gpu_norm_rope_values_and_errors():
    from sparse_attn_sharedkv_b200.rope import norm_rope
    x, cos, sin, w, _ = row_case(576, 64, 512, torch.float32, torch.bfloat16, 6, 5)
    x = x.view(6, 1, 576)
    x[1] = 0
    x[2, 0, 3] = float("nan")
    x[3, 0, 575] = float("inf")
    pos = torch.tensor([0, 1, 2, 3, 4096, -1]).cuda()
    y = norm_rope(x, pos, cos, sin, norm_dim=512, norm_weight=w)
    assert torch.equal(y[1], torch.zeros_like(y[1]))
    assert y[2, 0, :512].isnan().all() and y[2, 0, 512:].isfinite().all()
    assert y[3, 0, :574].isfinite().all() and not y[3, 0, 574:].isfinite().all()
    assert torch.equal(y[4:], torch.zeros_like(y[4:]))
    with pytest.raises(RuntimeError, match="outside the tables"):
        norm_rope(x, pos, cos, sin, norm_dim=512, check_errors=True)
    norm_rope(x[:4], pos[:4], cos, sin, norm_dim=512, check_errors=True)
    empty = norm_rope(x[:0], pos[:0], cos, sin)
    assert empty.shape == (0, 1, 576)
    for bad in (pos[:5], pos.float(), None):
        with pytest.raises(ValueError, match="positions"):
            norm_rope(x, bad, cos, sin)
    with pytest.raises(ValueError, match="out must"):
        norm_rope(x, pos, cos, sin, out=torch.empty_like(x[:5]))
    with pytest.raises(ValueError, match="float32 tensor on"):
        norm_rope(x, pos, cos.cpu(), sin.cpu())


@pytest.mark.gpu
def test_gpu_norm_rope_graph_and_stream():
    from sparse_attn_sharedkv_b200.rope import norm_rope
    x, cos, sin, w, _ = row_case(576, 64, 512, torch.float32, torch.bfloat16, 64 * 16, 7)
    x = x.view(64, 16, 576)
    pos = torch.arange(64, dtype=torch.int32).cuda()
    kw = dict(norm_dim=512, norm_weight=w)
    y = norm_rope(x, pos, cos, sin, **kw)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        z = norm_rope(x, pos, cos, sin, **kw)
    side.synchronize()
    assert torch.equal(z, y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        z = norm_rope(x, pos, cos, sin, **kw)
    x.copy_(x.flip(0))
    pos.add_(5)
    graph.replay()
    assert torch.equal(z, norm_rope(x, pos, cos, sin, **kw)) and not torch.equal(z, y)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D, rope, norm, wt, inter", [ROWS[i] for i in (0, 1, 3, 6, 8, 10, 12)])
@pytest.mark.parametrize("B, bs, ratio", [(1, 64, 1), (5, 1, 4), (40, 5, 1), (1300, 64, 2)])
def test_gpu_append_norm_rope(D, rope, norm, wt, inter, dtype, B, bs, ratio):
    from sparse_attn_sharedkv_b200.kv_cache import append_paged_kv_norm_rope
    rng = np.random.default_rng(B + bs)
    add = rng.integers(0, 4 if B > 100 else 40, B)
    add[rng.integers(0, B)] += 1
    if B > 1:
        add[0] = add[-1] = 0  # empty first and last sequences
        add[1] += 1
    start = rng.integers(0, 200, B)
    cu = np.concatenate([[0], np.cumsum(add)])
    n, behind = int(cu[-1]), 3
    per = -(-int((start + add).max() + 1) // bs)
    blocks = B * per + 2
    table = rng.permutation(blocks)[:B * per].reshape(B, per).astype(np.int32)
    x, cos, sin, w, _ = row_case(D, rope, norm, wt, dtype, n + behind, B)
    batch = np.repeat(np.arange(B), add)
    logical = start[batch] + np.arange(n) - cu[batch]
    want, mag = reference(x[:n], torch.from_numpy(logical * ratio), cos, sin, norm, w, inter)
    pool0 = torch.full((blocks, bs, 1, D), 7.0, dtype=dtype, device="cuda")
    pool = pool0.clone()
    t = lambda a: torch.from_numpy(np.asarray(a)).to(torch.int32).cuda()
    kw = dict(norm_dim=norm, norm_weight=w, eps=EPS, interleaved=inter, cmp_ratio=ratio)
    assert append_paged_kv_norm_rope(pool, t(table), x, t(cu), t(start), cos, sin,
                                     check_errors=True, **kw) is None
    slots = torch.from_numpy(table[batch, logical // bs] * bs + logical % bs).long().cuda()
    flat = pool.view(-1, D)
    check(flat[slots], want, mag, dtype)
    flat[slots] = 7.0
    assert torch.equal(pool, pool0)  # nothing else was written, the rows behind included


@pytest.mark.gpu
def test_gpu_append_norm_rope_skips_and_reports():
    from sparse_attn_sharedkv_b200.kv_cache import append_paged_kv_norm_rope
    x, cos, sin, w, _ = row_case(576, 64, 512, torch.float32, torch.bfloat16, 6, 9, 100)
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32).cuda()
    kw = dict(norm_dim=512, norm_weight=w, check_errors=True)

    def run(start, table, ratio=1):
        pool = torch.zeros(4, 4, 576, dtype=torch.bfloat16, device="cuda")
        e = append_paged_kv_norm_rope(pool, i32(table), x, i32(0, 6), i32(start), cos, sin,
                                      cmp_ratio=ratio, **kw)
        return e, pool.float().abs().sum(-1).view(-1).nonzero().flatten().tolist()

    assert run(2, [1, 0, 3]) == (None, [0, 1, 2, 3, 6, 7])
    e, slots = run(2, [1, -1, 3])          # rows 2..5 on the unmapped page
    assert e[:2] == [6, 50] and 2 <= e[2] <= 5 and slots == [6, 7]
    e, slots = run(2, [1, 4, 3])           # a page id outside the pool
    assert e[:2] == [6, 50] and slots == [6, 7]
    e, slots = run(10, [2, 1, 0])          # past the table
    assert e[:2] == [6, 50] and slots == [2, 3]
    e, slots = run(-2, [2, 1, 0])          # before the sequence
    assert e[:2] == [6, 50] and slots == [8, 9, 10, 11]
    e, slots = run(0, [2, 1, 0], 33)       # rows 4, 5 at rotation positions 132, 165
    assert e[:2] == [6, 51] and e[2] in (4, 5) and slots == [8, 9, 10, 11]


@pytest.mark.gpu
def test_gpu_plain_append_is_the_transform_of_nothing():
    # A norm weight of one and angles of zero on rows whose mean square is one: the copy.
    from sparse_attn_sharedkv_b200.kv_cache import append_paged_kv, append_paged_kv_norm_rope
    g = torch.Generator().manual_seed(1)
    x = torch.where(torch.rand(70, 576, generator=g) < 0.5, -1.0, 1.0).to(torch.bfloat16).cuda()
    table = torch.tensor([[3, 0, 2], [1, 5, 4]], dtype=torch.int32).cuda()
    cu = torch.tensor([0, 50, 70], dtype=torch.int32).cuda()
    start = torch.tensor([60, 7], dtype=torch.int32).cuda()
    cos, sin = torch.ones(256, 32).cuda(), torch.zeros(256, 32).cuda()
    a = torch.zeros(6, 64, 1, 576, dtype=torch.bfloat16).cuda()
    b = a.clone()
    append_paged_kv(a, table, x, cu, start)
    append_paged_kv_norm_rope(b, table, x, cu, start, cos, sin, norm_dim=512, eps=0.0)
    assert torch.equal(a, b)


