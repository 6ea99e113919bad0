"""The first call of a process to each operator before the attention, inside a graph capture."""

import os
import subprocess
import sys

import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

_SETUP = """
import torch
from sparse_attn_sharedkv_b200 import indexer, kv_cache, rope

g = torch.Generator().manual_seed(3)
rnd = lambda *s: torch.randn(*s, generator=g).to(torch.bfloat16).cuda()
i32 = lambda v: torch.tensor(v, dtype=torch.int32).cuda()
x, rows, pool = rnd(3, 16, 576), rnd(3, 576), torch.zeros(8, 64, 1, 576).to(torch.bfloat16).cuda()
cos, sin = torch.randn(512, 32, generator=g).cuda(), torch.randn(512, 32, generator=g).cuda()
table, cu = i32([[0, 1], [2, 3], [4, 5]]), i32([0, 1, 2, 3])
start = pos = i32([5, 6, 70])
qi, wi, keys = rnd(3, 64, 128), torch.randn(3, 64, generator=g).cuda(), rnd(8, 64, 1, 128)
scores = torch.randn(3, {cols}, generator=g).cuda()
kw = dict(key_pool=keys, block_table=table, cu_seqlens_q=cu, seqused_kv=i32([6, 7, 71]))

def append():
    kv_cache.append_paged_kv_norm_rope(pool, table, rows, cu, start, cos, sin, norm_dim=512)
    return pool

call = {call}
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    first = call()
first.zero_()
graph.replay()
first = first.clone()
pool.zero_()
assert torch.equal(first, call()) and bool((first != 0).any())
"""

CALLS = {
    "norm_rope": ("lambda: rope.norm_rope(x, pos, cos, sin, norm_dim=512)", 100),
    "append": ("append", 100),
    "index_scores": ("lambda: indexer.index_scores(qi, wi, **kw)", 100),
    "select_topk": ("lambda: indexer.select_topk(scores, 40)", 100),
    "select_topk_cluster": ("lambda: indexer.select_topk(scores, 40)", 40000),
    "select_topk_long": ("lambda: indexer.select_topk(scores, 40)", 270000),
    "select_keys": ("lambda: indexer.select_keys(qi, wi, topk=40, **kw)", 100),
}


@pytest.mark.gpu
@pytest.mark.parametrize("name", CALLS)
def test_gpu_first_call_is_captured(name):
    call, cols = CALLS[name]
    done = subprocess.run([sys.executable, "-c", _SETUP.format(call=call, cols=cols)], cwd=REPO,
                          env={**os.environ, "PYTHONPATH": REPO}, capture_output=True, text=True,
                          timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]
