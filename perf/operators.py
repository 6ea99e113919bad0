"""Measured cases of the operators between the projections and the attention: norm and rotation
of query heads, the normed and rotated append to a paged cache, the index scores of a query
against the index keys of a paged cache, and the top-k selection of the positions the attention
reads.

``own`` false: plain torch forms in 32 bits.  ``own`` true: the calls a user makes.
"""

import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
_EPS = 1e-6
_MAX_POS = 160_000  # past the furthest position of a case


def listed():
    return [
        # Queries of a two-sequence decode step: the smallest call, latency only.
        dict(name="norm_rope_decode_b2_h16", op="norm_rope", T=2, H=16, D=576, rope=64, norm=512,
             weight=True, interleaved=True, inverse=False, dtype="bf16"),
        # Queries of a ragged prompt batch (odd token count), norm over the whole head without a
        # weight, rotation by halves.
        dict(name="norm_rope_prompts_t7681_h64", op="norm_rope", T=7681, H=64, D=512, rope=64,
             norm=512, weight=False, interleaved=False, inverse=False, dtype="fp16"),
        # Queries of a long prompt chunk at the widest head layout.
        dict(name="norm_rope_prefill_t8192_h128", op="norm_rope", T=8192, H=128, D=576, rope=64,
             norm=512, weight=True, interleaved=True, inverse=False, dtype="bf16"),
        # One new row for each of 64 decoding sequences.
        dict(name="append_decode_b64", op="append", B=64, new="one", most=1, kv=8192, bs=64, D=576,
             rope=64, norm=512, weight=True, interleaved=True, ratio=1, dtype="bf16"),
        # Compressed rows (one for four tokens) of ragged chunks, some empty, into small pages.
        dict(name="append_ragged_b37_ratio4", op="append", B=37, new="ragged", most=301, kv=1000,
             bs=16, D=512, rope=64, norm=512, weight=True, interleaved=False, ratio=4,
             dtype="fp16"),
        # The rows of 8 prompts of 4096 tokens.
        dict(name="append_prefill_8x4096", op="append", B=8, new="all", most=4096, kv=0, bs=64,
             D=576, rope=64, norm=512, weight=True, interleaved=True, ratio=1, dtype="bf16"),
        # A few tokens of three sequences, odd head count and width, small pages.
        dict(name="scores_small_b3_h24", op="scores", B=3, q="ragged", most=3, kv_low=1500,
             kv_high=4097, H=24, D=96, bs=16, ratio=1, dtype="fp16"),
        # One token of each of 256 long sequences against a 4x-compressed cache.
        dict(name="scores_decode_b256_ratio4", op="scores", B=256, q="all", most=1, kv_low=131072,
             kv_high=131072, H=64, D=128, bs=64, ratio=4, dtype="bf16"),
        # 8 prompts of 4096 tokens, every token against the keys before it.
        dict(name="scores_prefill_8x4096", op="scores", B=8, q="all", most=4096, kv_low=4096,
             kv_high=4096, H=64, D=128, bs=64, ratio=1, dtype="bf16"),
        # Two decoding sequences.
        dict(name="topk_small_b2_k512", op="topk", rows=2, N=4097, low=4000, K=512, causal=False,
             ties=True),
        # 64 decoding sequences of 8192 to 32768 keys.
        dict(name="topk_decode_b64_k2048", op="topk", rows=64, N=32768, low=8192, K=2048,
             causal=False, ties=False),
        # 8 prompts of 4096 tokens: each row has the keys before its token.
        dict(name="topk_prefill_8x4096_k2048", op="topk", rows=32768, N=4096, low=1, K=2048,
             causal=True, ties=False),
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["norm_rope", "append", "scores", "topk"])
    if op in ("norm_rope", "append"):
        D = rng.choice([64, 128, 200, 512, 576])
        row = dict(op=op, D=D, rope=rng.choice([32, 64]), norm=rng.choice([0, D, D - 64 or D, 40]),
                   weight=rng.random() < 0.7, interleaved=rng.random() < 0.5,
                   dtype=rng.choice(["bf16", "fp16"]))
        if op == "norm_rope":
            H = _log(rng, 1, 128)
            row.update(H=H, inverse=rng.random() < 0.25)
            row["T"] = _log(rng, 1, max(2, 8192 * 128 // (4 * H)))
        else:
            B = _log(rng, 1, 200)
            row.update(B=B, new=rng.choice(["one", "ragged"]), most=_log(rng, 1, 30000 // B + 1),
                       kv=_log(rng, 1, 8192), bs=rng.choice([1, 5, 16, 64, 100, 128]),
                       ratio=rng.choice([1, 4]))
        return row
    if op == "scores":
        B, D = _log(rng, 1, 64), rng.choice([32, 64, 96, 128])
        H = rng.choice([1, 8, 16, 24, 32, 64, 100, 128])
        ratio = rng.choice([1, 4, 128])
        most = 1 if rng.random() < 0.4 else _log(rng, 1, 512)
        # B * most * H * keys stays well below the largest listed case's.
        keys = max(1, min(40000 // ratio, 4_000_000_000 // (B * most * H), 40_000_000 // (B * 16)))
        high = max(2, _log(rng, 1, keys) * ratio)
        return dict(op=op, B=B, q=rng.choice(["all", "ragged"]), most=most,
                    kv_low=max(ratio, high // 4), kv_high=high, H=H, D=D,
                    bs=rng.choice([3, 16, 48, 64, 128]), ratio=ratio,
                    dtype=rng.choice(["bf16", "fp16"]))
    N = _log(rng, 64, 131072)
    K = min(rng.choice([1, 64, 500, 512, 1000, 2048]), N // 4)
    return dict(op=op, rows=_log(rng, 1, max(2, 60_000_000 // (N + K))), N=N,
                low=rng.choice([N // 2, N]), K=K, causal=rng.random() < 0.4,
                ties=rng.random() < 0.4)


# ---- lengths of a case: by the case alone, so that work() knows them ----

def _spread(case, count, low, high):
    rng = random.Random("%d %d %d" % (count, low, high))
    return [rng.randint(low, high) for _ in range(count)]


def _new_rows(case):
    B, most = case["B"], case["most"]
    if case["new"] == "one":
        return [1] * B
    if case["new"] == "all":
        return [most] * B
    got = _spread(case, B, 0, most)
    got[0] = max(got[0], 1)
    return got


def _q_lens(case):
    return [case["most"]] * case["B"] if case["q"] == "all" else _spread(case, case["B"], 1,
                                                                         case["most"])


def _kv_lens(case):
    # A sequence holds at least its own new tokens.
    return [max(n, q) for n, q in zip(_spread(case, case["B"], case["kv_low"], case["kv_high"]),
                                      _q_lens(case))]


def _thresholds(case):
    """Keys each token sees: floor((kv - q + s + 1) / ratio)."""
    return [(kv - q + s + 1) // case["ratio"] for kv, q in zip(_kv_lens(case), _q_lens(case))
            for s in range(q)]


def _columns(case):
    return max(1, max(_kv_lens(case)) // case["ratio"])


def _row_lens(case):
    rows, N, low = case["rows"], case["N"], case["low"]
    if case["causal"]:
        return [N - (rows - 1 - i) % N for i in range(rows)]
    return _spread(case, rows, min(low, N), N)


# ---- inputs ----

def _angles(rope, device):
    """cos, sin [positions, rope / 2] of a 10000-based rotation, angles in 64 bits."""
    freq = 10000.0 ** (-torch.arange(0, rope, 2, dtype=torch.float64, device=device) / rope)
    angle = torch.arange(_MAX_POS, dtype=torch.float64, device=device)[:, None] * freq
    return angle.cos().float(), angle.sin().float()


def _row_setup(case, g, s):
    dev = "cuda"
    s["cos"], s["sin"] = _angles(case["rope"], dev)
    s["norm"] = case["norm"]
    s["weight"] = None
    if case["weight"] and case["norm"]:
        s["weight"] = 1 + 0.2 * torch.randn(case["norm"], generator=g, device=dev)
    s["interleaved"], s["inverse"] = case["interleaved"], case.get("inverse", False)


def _pages(g, B, per):
    """Block tables over randomly placed pages, each sequence with pages of its own."""
    return torch.randperm(B * per, generator=g, device="cuda").to(torch.int32).view(B, per)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dev, op = "cuda", case["op"]
    s = {"op": op}

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=dev, dtype=torch.bfloat16
                           if case["dtype"] == "bf16" else torch.float16)

    if op == "norm_rope":
        T, H, D = case["T"], case["H"], case["D"]
        s["x"] = randn(T, H, D)
        s["positions"] = torch.randint(0, _MAX_POS, (T,), generator=g, device=dev,
                                       dtype=torch.int32)
        _row_setup(case, g, s)
    elif op == "append":
        B, D, bs = case["B"], case["D"], case["bs"]
        new = _new_rows(case)
        s["rows"] = randn(sum(new), D)
        s["cu"] = torch.tensor([sum(new[:b]) for b in range(B + 1)], dtype=torch.int32, device=dev)
        s["start"] = torch.randint(0, case["kv"] + 1, (B,), generator=g, device=dev,
                                   dtype=torch.int32)
        per = -(-(case["kv"] + max(new)) // bs)
        s["table"] = _pages(g, B, per)
        s["pool"] = torch.zeros(B * per, bs, 1, D, device=dev, dtype=_DTYPES[case["dtype"]])
        s["ratio"] = case["ratio"]
        _row_setup(case, g, s)
    elif op == "scores":
        B, H, D, bs = case["B"], case["H"], case["D"], case["bs"]
        q_lens, kv_lens, N = _q_lens(case), _kv_lens(case), _columns(case)
        T = sum(q_lens)
        s["q"] = randn(T, H, D)
        s["w"] = torch.randn(T, H, generator=g, device=dev) * (H * D) ** -0.5
        per = -(-N // bs)
        s["table"] = _pages(g, B, per)
        s["pool"] = randn(B * per, bs, 1, D)
        s["cu"] = torch.tensor([sum(q_lens[:b]) for b in range(B + 1)], dtype=torch.int32,
                               device=dev)
        s["kv"] = torch.tensor(kv_lens, dtype=torch.int32, device=dev)
        s["ratio"], s["N"], s["longest"] = case["ratio"], N, max(q_lens)
    else:
        rows, N = case["rows"], case["N"]
        # Weighted sums of rectified products: a skewed bulk with a tail.
        x = torch.randn(rows, N, generator=g, device=dev)
        x = torch.where(x > 0, x * x, 0.1 * x)
        s["scores"] = x.to(torch.bfloat16).float() if case["ties"] else x
        s["lengths"] = torch.tensor(_row_lens(case), dtype=torch.int32, device=dev)
        s["K"] = case["K"]
    return s


# ---- plain forms ----

def _plain_rows(x, positions, s):
    """x [..., D] normed over its first columns, the last ones rotated; fp32."""
    x = x.float()
    D, n = x.shape[-1], s["norm"]
    if n:
        y = x[..., :n] * torch.rsqrt(x[..., :n].square().mean(-1, keepdim=True) + _EPS)
        if s["weight"] is not None:
            y = y * s["weight"]
        x = torch.cat([y, x[..., n:]], -1)
    cos, sin = s["cos"][positions.long()], s["sin"][positions.long()]
    half = cos.shape[-1]
    if x.dim() == 3:
        cos, sin = cos[:, None], sin[:, None]
    if s["inverse"]:
        sin = -sin
    keep, rot = x[..., :D - 2 * half], x[..., D - 2 * half:]
    if s["interleaved"]:
        a, b = rot[..., 0::2], rot[..., 1::2]
        rot = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = rot[..., :half], rot[..., half:]
        rot = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([keep, rot], -1)


def _batch_of(cu, total):
    token = torch.arange(total, device=cu.device)
    batch = torch.searchsorted(cu[1:].long(), token, right=True)
    return batch, token - cu.long()[batch]


def _plain_append(s):
    rows, pool = s["rows"], s["pool"]
    batch, i = _batch_of(s["cu"], rows.shape[0])
    p = s["start"].long()[batch] + i
    bs = pool.shape[1]
    y = _plain_rows(rows, p * s["ratio"], s).to(pool.dtype)
    pool[s["table"].long()[batch, p // bs], p % bs, 0] = y
    return pool


def _plain_scores(s):
    q, w, pool, N = s["q"], s["w"], s["pool"], s["N"]
    T, H, D = q.shape
    B, bs, S = s["kv"].numel(), pool.shape[1], s["longest"]
    j = torch.arange(N, device=q.device)
    keys = pool.view(-1, D)[s["table"].long()[:, j // bs] * bs + j % bs].float()
    batch, i = _batch_of(s["cu"], T)
    at = (s["cu"].long()[:-1, None] + torch.arange(S, device=q.device)).clamp(max=T - 1)
    dots = torch.bmm(q[at].float().view(B, S * H, D), keys.transpose(1, 2)).clamp_min_(0)
    out = torch.bmm(w[at].view(B * S, 1, H), dots.view(B * S, H, N)).view(B, S, N)[batch, i]
    q_len = (s["cu"][1:] - s["cu"][:-1]).long()
    seen = (s["kv"].long()[batch] - q_len[batch] + i + 1) // s["ratio"]
    return out.masked_fill_(j >= seen[:, None], float("-inf"))


def _plain_topk(s):
    x, K = s["scores"], s["K"]
    rows, N = x.shape
    x = x.masked_fill(torch.arange(N, device=x.device) >= s["lengths"][:, None], float("-inf"))
    best = torch.sort(x, dim=1, descending=True, stable=True)
    at = best.indices[:, :K].masked_fill_(best.values[:, :K] == float("-inf"), N)
    at = at.sort(dim=1).values
    at = at.masked_fill_(at == N, -1).to(torch.int32)
    if K > N:
        at = torch.cat([at, at.new_full((rows, K - N), -1)], 1)
    return at[:, None]


def run(s):
    op = s["op"]
    if own:
        from sparse_attn_sharedkv_b200 import indexer, kv_cache, rope
        if op == "norm_rope":
            return rope.norm_rope(s["x"], s["positions"], s["cos"], s["sin"], norm_dim=s["norm"],
                                  norm_weight=s["weight"], eps=_EPS,
                                  interleaved=s["interleaved"], inverse=s["inverse"])
        if op == "append":
            kv_cache.append_paged_kv_norm_rope(
                s["pool"], s["table"], s["rows"], s["cu"], s["start"], s["cos"], s["sin"],
                norm_dim=s["norm"], norm_weight=s["weight"], eps=_EPS,
                interleaved=s["interleaved"], cmp_ratio=s["ratio"])
            return s["pool"]
        if op == "scores":
            return indexer.index_scores(s["q"], s["w"], key_pool=s["pool"],
                                        block_table=s["table"], cu_seqlens_q=s["cu"],
                                        seqused_kv=s["kv"], cmp_ratio=s["ratio"],
                                        max_keys=s["N"])
        return indexer.select_topk(s["scores"], s["K"], lengths=s["lengths"])
    if op == "norm_rope":
        return _plain_rows(s["x"], s["positions"], s).to(s["x"].dtype)
    return {"append": _plain_append, "scores": _plain_scores, "topk": _plain_topk}[op](s)


# ---- the definitions in 64 bits ----

def _exact_rows(x, positions, s):
    """Row by row of the definition: a complex product for each rotated pair."""
    y = x.double().clone()
    n, half, D = s["norm"], s["cos"].shape[1], x.shape[-1]
    if n:
        scale = 1 / torch.sqrt((y[..., :n] ** 2).sum(-1, keepdim=True) / n + _EPS)
        y[..., :n] *= scale
        if s["weight"] is not None:
            y[..., :n] *= s["weight"].double()
    turn = torch.complex(s["cos"].double(), s["sin"].double())[positions.long()]
    if s["inverse"]:
        turn = turn.conj()
    if x.dim() == 3:
        turn = turn[:, None]
    tail = y[..., D - 2 * half:]
    if s["interleaved"]:
        z = torch.complex(tail[..., 0::2].contiguous(), tail[..., 1::2].contiguous()) * turn
        tail[..., 0::2], tail[..., 1::2] = z.real, z.imag
    else:
        z = torch.complex(tail[..., :half].contiguous(), tail[..., half:].contiguous()) * turn
        tail[..., :half], tail[..., half:] = z.real, z.imag
    return y


def exact(case, seed):
    op = case["op"]
    if op == "topk":
        return None
    s = prepare(case, seed)
    if op == "norm_rope":
        if s["x"].numel() > 400_000_000:
            return None
        return _exact_rows(s["x"], s["positions"], s)
    if op == "append":
        rows, cu, bs = s["rows"], s["cu"].tolist(), case["bs"]
        starts, table = s["start"].tolist(), s["table"].cpu()
        places, positions = [], []
        for b in range(case["B"]):
            for i in range(cu[b + 1] - cu[b]):
                p = starts[b] + i
                places.append(int(table[b, p // bs]) * bs + p % bs)
                positions.append(p * case["ratio"])
        pool = s["pool"].double()
        y = _exact_rows(rows, torch.tensor(positions, device=rows.device), s)
        pool.view(-1, case["D"])[torch.tensor(places, device=rows.device)] = y
        return pool
    N, bs, H, D = s["N"], case["bs"], case["H"], case["D"]
    out = torch.full((s["q"].shape[0], N), float("-inf"), dtype=torch.float64, device="cuda")
    seen = torch.tensor(_thresholds(case), device="cuda")
    cu = s["cu"].tolist()
    for b in range(case["B"]):
        keys = s["pool"][s["table"][b].long()].reshape(-1, D)[:N].double()
        for t in range(cu[b], cu[b + 1], 256):
            u = min(t + 256, cu[b + 1])
            total = torch.zeros(u - t, N, dtype=torch.float64, device="cuda")
            for h in range(H):
                total += s["w"][t:u, h, None].double() * torch.relu(s["q"][t:u, h].double()
                                                                    @ keys.T)
            valid = torch.arange(N, device="cuda") < seen[t:u, None]
            out[t:u] = torch.where(valid, total, out[t:u])
    return out


def work(case):
    op = case["op"]
    if op == "norm_rope":
        n = case["T"] * case["H"] * case["D"]
        return {"bytes": 4 * n + case["T"] * (4 + 4 * case["rope"]), "flops": 6 * n}
    if op == "append":
        rows = sum(_new_rows(case))
        return {"bytes": rows * (4 * case["D"] + 4 * case["rope"] + 4),
                "flops": 6 * rows * case["D"]}
    if op == "scores":
        seen = _thresholds(case)
        T, N, H, D = len(seen), _columns(case), case["H"], case["D"]
        keys = sum(kv // case["ratio"] for kv in _kv_lens(case))
        return {"bytes": 2 * D * (keys + T * H) + 4 * T * (H + N),
                "flops": sum(seen) * H * (2 * D + 2)}
    lens = _row_lens(case)
    return {"bytes": 4 * (sum(lens) + case["rows"] * (case["K"] + 1)), "flops": sum(lens)}
