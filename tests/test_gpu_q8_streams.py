"""Plans (of the 8-bit cache, and of the block) on streams other than the one they were made on."""
import pytest
import torch

import test_gpu_q8 as Q
from triton_b200 import ops

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _attend():
    q, kc, vc, ks, vs = Q._attend_inputs(1, 1, 8, 2, 64, 9000, 64, BF, 3)
    cache, _, _ = Q._cache(kc, vc, ks, vs, 64)
    q = q.cuda()
    return lambda: ops.AttentionQ8Plan(q, cache, torch.empty_like(q), kv_len=9000)


def _evict():
    k = torch.randn(1, 9000, 1, 64, device="cuda").to(BF)
    to = torch.empty(1, 500, 1, 64, dtype=BF, device="cuda")
    scores = torch.rand(1, 8, 9000, device="cuda")
    return lambda: ops.CacheEvictPlan((k, k), (to, to.clone()), scores, kv_len=9000, keep=500)


def _block():
    B, M, P, H, D = 1, 64, 2000, 8, 128
    q, o = (torch.randn(B, M, H, D, device="cuda").to(BF) for _ in range(2))
    k, v = (torch.randn(B, P + M, H, D, device="cuda").to(BF) for _ in range(2))
    return lambda: ops.BlockPlan("vanilla", B=B, M=M, P=P, Hq=H, Hkv=H, D=D, q=q, k_cache=k, v_cache=v, o=o, scale=D ** -0.5)


@pytest.mark.parametrize("make", [_attend, _evict, _block])
def test_scratch_of_a_dropped_plan_waits_for_the_stream_that_used_it(make):
    """Made on one stream, run on another that is still busy, dropped: the scratch is not handed out again meanwhile."""
    build = make()
    torch.cuda.synchronize()
    home, busy = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(home):
        plan = build()
        plan.run()                                 # (loads the kernels: the queued run below shall not wait for that)
    torch.cuda.synchronize()
    where, size = plan.args.workspace, plan.args.workspace_bytes
    assert size > 0
    with torch.cuda.stream(busy):
        torch.cuda._sleep(400_000_000)             # about 0.2 s
        plan.run()
    del plan
    with torch.cuda.stream(home):
        again = [torch.empty(size, dtype=torch.uint8, device="cuda") for _ in range(3)]
    still = not busy.query()
    Q._done()
    assert still, "the other stream was done too early for this test to tell"
    assert all(t.data_ptr() + size <= where or t.data_ptr() >= where + size for t in again)      # none reaches into it


def test_one_plan_on_several_streams_in_turn():
    q, kc, vc, ks, vs = Q._attend_inputs(2, 1, 8, 2, 128, 9100, 32, BF, 31)
    cache, _, _ = Q._cache(kc, vc, ks, vs, 32)
    qd, o = q.cuda(), torch.zeros(q.shape, dtype=BF, device="cuda")
    alone = ops.attention_q8(qd, cache, kv_len=9100)
    plan = ops.AttentionQ8Plan(qd, cache, o, kv_len=9100)
    torch.cuda.synchronize()
    for _ in range(3):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            o.zero_()
            plan.run()
            got = o.clone()
        s.synchronize()
        assert torch.equal(got, alone)
    Q._done()


@pytest.mark.parametrize("S", [600, 9000])
def test_a_captured_plan_with_scratch_of_its_own(S):
    """Made outside, captured on the capture's stream, replayed on another, graph and plan dropped: what comes after is sound."""
    q, kc, vc, ks, vs = Q._attend_inputs(2, 1, 8, 2, 64, S, 64, BF, 37)
    cache, _, _ = Q._cache(kc, vc, ks, vs, 64)
    qd, o, w = q.cuda(), torch.zeros(q.shape, dtype=BF, device="cuda"), torch.zeros(2, 2, S, device="cuda")
    want_w = torch.zeros_like(w)
    want = ops.attention_q8(qd, cache, kv_len=S, weight=want_w)
    plan = ops.AttentionQ8Plan(qd, cache, o, kv_len=S, weight=w)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan.run()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(3):
            graph.replay()
    Q._done()
    assert torch.equal(o, want) and torch.equal(w, want_w)
    del graph, plan
    other = [torch.full((1 << 20,), 7, dtype=torch.uint8, device="cuda") for _ in range(8)]
    again = ops.attention_q8(qd, cache, kv_len=S)
    Q._done()
    assert torch.equal(again, want) and all(bool((t == 7).all()) for t in other)
