"""Layers of drafted tokens and their kept rows on several streams and from several threads."""

import threading

import pytest
import torch

from falcon_perception_amd import ops
from tests.draft_cases import DraftBatch, random_tree

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def layer_set(seed, B, S):
    """Everything that a layer of drafts and its kept rows take, with buffers of its own."""
    gen = torch.Generator().manual_seed(seed)
    case = DraftBatch(seed, [], [(-1, 30 + 40 * b, random_tree(gen, S, 1 + b % 3)) for b in range(B)], Hq=8, Hc=2, D=64, P=32, dtype=BF16).on()
    case.pool_d.nan_to_num_(0.0)
    shape = dict(q_heads=8, cached_heads=2, head_dim=64)
    case.plan = torch.empty(ops.shared_decode_plan_bytes(B, S, **shape), dtype=torch.uint8, device="cuda")
    case.ws = torch.empty(ops.shared_decode_workspace_bytes(B, S, **shape), dtype=torch.uint8, device="cuda")
    case.start = case.pool_d.clone()
    case.path = torch.full((B, S), -1, dtype=torch.int32)
    for b in range(B):
        n = 1 + b % (S - 1)
        case.path[b, :n] = torch.tensor(sorted(torch.randperm(S, generator=gen)[:n].tolist()), dtype=torch.int32)
    case.path_d = case.path.cuda()

    def run():
        case.pool_d.copy_(case.start)
        tree = ops.draft_tree(case.parents_d, case.cached_d)
        ops.tree_decode_plan(case.batch_idx_d, tree, case.table_d, q_heads=8, cached_heads=2, head_dim=64, max_context=case.columns * 32, plan=case.plan)
        out, lse = ops.paged_decode_tree(case.q_d, case.pool_d[0], case.pool_d[1], case.table_d, case.batch_idx_d, tree, 32, case.columns * 32,
                                         plan=case.plan, workspace=case.ws)
        ops.keep_rows(case.pool_d, case.table_d, case.batch_idx_d, case.cached_d, case.path_d, 32)
        return out, lse, case.pool_d

    return run


def test_layers_on_several_streams():
    """Two graphs of a layer and its kept rows, replayed on two streams at once, and an eager layer on a third: buffers of each one's own."""
    runs = [layer_set(60 + i, 5 + i, 7) for i in range(3)]
    want = [[t.clone() for t in run()] for run in runs]
    torch.cuda.synchronize()
    graphs, results = [], []
    for run in runs[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            results.append(run())
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(12):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        with torch.cuda.stream(streams[2]):
            third = runs[2]()
        torch.cuda.synchronize()
        for got, w in zip([*results, third], want):
            for x, y in zip(got, w):
                assert torch.equal(x, y)


def test_layers_from_several_threads():
    runs = [layer_set(70 + i, 4, 6) for i in range(2)]
    want = [[t.clone() for t in run()] for run in runs]
    torch.cuda.synchronize()
    wrong = []

    def work(run, w):
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            for _ in range(60):
                got = run()
                st.synchronize()
                if not all(torch.equal(x, y) for x, y in zip(got, w)):
                    wrong.append(1)
                st.synchronize()

    threads = [threading.Thread(target=work, args=a) for a in zip(runs, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
