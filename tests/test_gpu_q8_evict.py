"""Eviction from a cache: sums of score heads whose order shows, and rows at the borders of how the work is divided."""
import pytest
import torch

import q8_oracle as O
import test_gpu_q8 as Q
from triton_b200 import ops

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.mark.parametrize("Hs,Hkv,n", [(21, 3, 9001), (5, 1, 8000), (9, 3, 12000), (71, 1, 3000), (142, 2, 1111)])
def test_sums_of_scores_that_cancel_are_the_same_with_and_without_scratch(Hs, Hkv, n):
    """Scores of either sign and sizes 1e20 apart: their 64-bit sums depend on the order, which is the same in both kernels."""
    B, keep = 2, 300
    g = torch.Generator().manual_seed(53)
    scores = torch.randn(B, Hs, n, generator=g)
    scores *= torch.tensor([1.0, 1e10, 1e20])[torch.randint(0, 3, scores.shape, generator=g)]
    half = Hs // Hkv // 2                          # within a group: large ones of both signs, which cancel
    for h in range(Hkv):
        a = h * (Hs // Hkv)
        scores[:, a + half:a + 2 * half] = -scores[:, a:a + half] * (1 + 2.0 ** -20 * torch.randint(0, 2, (B, half, n), generator=g))
    k = torch.randn(B, n, Hkv, 64, generator=g).to(BF).cuda()
    outs = []
    for scratch in (True, False):
        to, sout = torch.zeros(B, keep, Hkv, 64, dtype=BF, device="cuda"), torch.zeros(B, Hkv, keep, device="cuda")
        plan = ops.CacheEvictPlan((k, k), (to, to.clone()), scores.cuda(), kv_len=torch.tensor([n, n - 7], dtype=torch.int32).cuda(),
                                  keep=keep, recent=7, first=2, scores_out=sout)
        assert plan.args.workspace_bytes == 4 * B * Hkv * n
        if not scratch:
            plan.args.workspace = None
        plan.run()
        Q._done()
        outs.append((plan.idx, sout, to))
    assert all(torch.equal(a, c) for a, c in zip(*outs))


@pytest.mark.parametrize("G", [1, 2, 3, 4, 5, 6, 7, 8, 9, 31])
def test_group_sums_of_few_heads(G):
    """Whole numbers, so that every order gives the same sum: each head counted once, however many there are."""
    B, Hkv, n, keep = 1, 2, 500, 90
    g = torch.Generator().manual_seed(G)
    scores = torch.randint(-1000, 1000, (B, Hkv * G, n), generator=g).float()
    k = torch.randn(B, n, Hkv, 64, generator=g).to(BF).cuda()
    to, sout = torch.zeros(B, keep, Hkv, 64, dtype=BF, device="cuda"), torch.zeros(B, Hkv, keep, device="cuda")
    idx = ops.cache_evict((k, k), (to, to.clone()), scores.cuda(), kv_len=n, keep=keep, recent=3, scores_out=sout)
    Q._done()
    kept, w = O.select(scores[0], n, keep, 3, 0, G)
    for h in range(Hkv):
        assert idx[0, h].tolist() == kept[h] and torch.equal(sout[0, h].cpu(), w[h][kept[h]])
