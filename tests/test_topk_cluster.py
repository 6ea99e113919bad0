"""Clusters of the top-k selection: shared memory of another block is reached for only once
every block of the cluster is known to run."""

import os
import re

import numpy as np
import pytest
import torch

from sparse_attn_sharedkv_b200 import indexer
from sparse_attn_sharedkv_b200.build import CSRC

from .test_indexer import KINDS, topk_reference, topk_rows

# What touches another block's shared memory, itself or (for rows of several blocks) inside.
_PEER = re.compile(r"\b(peer_\w+|row_reduce|find_bin|count_before|add_entry|list_threshold|"
                   r"select_general)\s*(<[^<>()]*>)?\s*\(")
_ARRIVE = re.compile(r"\bpeers_arrive\s*<\s*C\s*>\s*\(\)")
_WAIT = re.compile(r"\bpeers_wait\s*<\s*C\s*>\s*\(\)")


def cluster_kernels():
    """(name, body) of each kernel of the file that is launched as clusters."""
    with open(os.path.join(CSRC, "sas_topk.cu")) as f:
        text = re.sub(r"//[^\n]*", "", f.read())
    for m in re.finditer(r"__global__[^;{]*?__cluster_dims__\s*\([^;{]*?(\w+)\s*\([^;{]*?\)\s*\{",
                         text, re.S):
        depth, end = 1, m.end()
        while depth:
            depth += {"{": 1, "}": -1}.get(text[end], 0)
            end += 1
        yield m.group(1), text[m.end():end]


# ---- without a GPU ----

def test_cluster_kernels_wait_for_their_peers():
    kernels = dict(cluster_kernels())
    assert set(kernels) == {"topk_kernel", "topk_long_kernel"}
    for name, body in kernels.items():
        arrive, wait, peer = (p.search(body) for p in (_ARRIVE, _WAIT, _PEER))
        assert arrive and wait and peer, name
        assert arrive.start() < wait.start() < peer.start(), name
        assert len(_ARRIVE.findall(body)) == len(_WAIT.findall(body)) == 1, name
        # The one way out before the arrival is that of empty rows, which all blocks of a row
        # take; between the arrival and the wait only rows of one block leave.
        assert len(re.findall(r"\breturn\b", body[:arrive.start()])) == 1, name
        for m in re.finditer(r"[^\n]*\breturn\b", body[arrive.end():wait.start()]):
            assert "C == 1" in m.group(), (name, m.group())


def test_cluster_barriers_take_diverged_warps():
    # Loops whose length differs between the lanes of a warp end right before some of them.
    with open(os.path.join(CSRC, "sas_topk.cu")) as f:
        barriers = re.findall(r"barrier\.cluster\.[\w.]+", f.read())
    assert len(barriers) == 4 and not any("aligned" in b for b in barriers)


# ---- on a GPU ----

@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows, N, K", [(24, 20000, 600), (24, 50000, 2048), (24, 100000, 2048),
                                        (24, 150000, 1000), (24, 300000, 2048)])
def test_gpu_clusters_of_empty_short_and_whole_rows(rows, N, K, kind):
    # Rows of all kinds of lengths in turn, more of them than clusters of eight run at once.
    g = torch.Generator().manual_seed(N + K)
    x = topk_rows(kind, 5, N, g)
    lengths = torch.randint(0, N + 1, (rows,), generator=g, dtype=torch.int32)
    lengths[::3] = torch.tensor([0, 1, 7, K, K + 1, N, N - 1])[torch.arange(len(lengths[::3])) % 7]
    at = torch.arange(rows) % 5
    d = x.cuda()[at.cuda()]
    got = indexer.select_topk(d, K, lengths=lengths.cuda())
    x = x.numpy()
    want = np.concatenate([topk_reference(x[int(a)][None], K, [int(n)])
                           for a, n in zip(at, lengths)])
    assert np.array_equal(got[:, 0].cpu().numpy(), want)
    assert torch.equal(indexer.select_topk(d, K, lengths=lengths.cuda()), got)
