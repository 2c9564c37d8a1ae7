"""Attention over the 8-bit cache at the ends of what its scales, queries and probabilities may be, in both of its kernels
(few rows per kv head; many)."""
import math

import pytest
import torch

import q8_oracle as O
import test_gpu_q8 as Q
from triton_b200 import ops

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def _call(q, kc, vc, ks, vs, lens, block, causal=True, weigh=False, **kw):
    """One call and its result in 64 bits."""
    B, M, Hq, D = q.shape
    Hkv, S = kc.shape[1:3]
    r = O.attend(q, Q._values(kc, ks, block), Q._values(vc, vs, block), lens, causal, D ** -0.5)
    cache, _, _ = Q._cache(kc, vc, ks, vs, block)
    o, lse = torch.zeros(B, M, Hq, D, dtype=q.dtype, device="cuda"), torch.zeros(B, Hq, M, device="cuda")
    w = torch.zeros(B, Hkv, S, device="cuda") if weigh else None
    ops.attention_q8(q.cuda(), cache, o, kv_len=torch.tensor(lens, dtype=torch.int32).cuda(), causal=causal, lse=lse, weight=w, **kw)
    Q._done()
    return o, lse, w, r


# --------------------------------------------------------------------------------------- scales of the values far apart

FAR = [
    # M, Hq, Hkv, D, n, block, dtype, weigh
    (1, 4, 2, 128, 200, 16, BF, True),           # a cluster for each unit
    (2, 4, 2, 64, 900, 64, BF, True),
    (1, 4, 2, 128, 9000, 128, BF, True),         # pieces, merged
    (9, 4, 1, 64, 5000, 32, BF, True),           # 36 rows: weights by threads that share the rows
    (40, 4, 2, 128, 300, 16, BF, False),         # tensor-core kernel
    (70, 4, 2, 64, 2000, 32, BF, False),         # ... its key blocks divided among CTAs
    (1, 4, 2, 128, 200, 16, HF, True),
    (40, 4, 2, 64, 300, 16, HF, False),
]


@pytest.mark.parametrize("low,high,order", [(2.0 ** -64, 2.0 ** 80, "mixed"), (2.0 ** -64, 2.0 ** 120, "mixed"), (2.0 ** -64, 2.0 ** 120, "rising"),
                                            (2.0 ** -64, 2.0 ** 120, "falling"), (0.0, 2.0 ** 40, "mixed"), (0.0, 2.0 ** 100, "rising")])
@pytest.mark.parametrize("M,Hq,Hkv,D,n,block,dt,weigh", FAR)
def test_value_scales_at_both_ends_of_their_range(M, Hq, Hkv, D, n, block, dt, weigh, low, high, order):
    """Blocks with the smallest scales keep their weight in the softmax beside blocks with the largest: mixed, the large ones last
    (what was summed moves to a larger maximum) and first."""
    if dt == HF:                                 # whose largest number bounds the scale
        low, high = (0.0, 2.0 ** 4) if low == 0.0 else (2.0 ** -64, 2.0 ** 5)
    q, kc, vc, ks, vs = Q._attend_inputs(1, M, Hq, Hkv, D, n, block, dt, 71)
    nblk = vs.shape[2]
    is_high = {"mixed": torch.arange(nblk) % 3 == 1, "rising": torch.arange(nblk) >= nblk // 2, "falling": torch.arange(nblk) < nblk // 2}[order]
    vs[:] = torch.where(is_high, high, low)
    if low == 0.0:
        vc[:, :, ~is_high.repeat_interleave(block)[:n]] = 0
    if high == 2.0 ** 120:                       # what an append leaves there: below 2^128 with its scale
        vc = ((vc.view(torch.float8_e4m3fn).float().clamp(-240, 240)).to(torch.float8_e4m3fn)).view(torch.uint8)
    o, lse, w, r = _call(q, kc, vc, ks, vs, [n], block, weigh=weigh)
    # Beside what _check counts: a maximum of size up to 128 + |t| has a step of 2^-16 (half of it in each of the exponents of a term, and
    # the same in lse), and a smallest term flushed at 2^-126 against a sum of 2^-96 or more, n of them at most
    extra = 2.0 ** -15 + n * 2.0 ** -30
    far = r["lse"].isfinite()
    ds = (D + 8) * 2.0 ** -23 * r["T"] + 2.0 ** -21
    e = (lse.double().cpu() - r["lse"]).abs()
    assert torch.equal(lse.cpu().double() == -math.inf, ~far)
    assert bool((e <= 1.5 * ds + 2.0 ** -21 * (1 + r["lse"].abs()) + extra)[far].all()), e[far].max().item()
    # o, each column against its own sum of p |v|, and against what a subnormal P' of fp16 loses: half a step, 2^-25, of at least 2^6
    # that the largest p vs has, times codes of up to 448
    top = Q._values(torch.full_like(vc, 0x38), vs, block).amax().item()
    tol, _ = Q._tolerance(r, q, dt, D)
    tol = tol + extra * r["A"] + (448 * n * 2.0 ** -31 * top if order != "mixed" else 0.0)
    e = (o.double().cpu() - r["o"]).abs()
    assert bool((e <= tol).all()), (e / tol).max().item()
    if weigh:
        e = (w.double().cpu() - r["weight"]).abs()
        rel = 2 * ds.amax().item() + 2.0 ** -23 * M * Hq // Hkv + 2.0 ** -20 + 2 * extra
        assert bool((e <= rel * r["weight"] + 1e-30).all()), (e / r["weight"].clamp_min(1e-30)).max().item()


@pytest.mark.parametrize("M,n,weigh", [(1, 70000, True), (40, 40000, False)])
def test_a_cache_of_zeros_with_scale_zero(M, n, weigh):
    """Values of 0 with a scale of 0 throughout, as a cache that was never filled holds them: the weights are those of the keys, and
    the sums of many large terms stay in range.  One query row, then 40 in the tensor-core kernel, where the keys behind the first
    block score 2^7.2 times as much as that one: under the 2^8 by which a score may pass the maximum in use."""
    D, block = 64, 128
    q = torch.zeros(1, M, 2, D)
    q[..., 0] = 1.0
    q[:, :, 1] *= -1.0
    q = q.to(BF)
    kc, vc = torch.zeros(1, 1, n, D, dtype=torch.uint8), torch.zeros(1, 1, n, D, dtype=torch.uint8)
    if M > 1:
        kc[0, 0, block:, 0] = torch.tensor(40.0).to(torch.float8_e4m3fn).view(torch.uint8).item()
    ks = torch.ones(1, 1, -(-n // block))
    vs = torch.zeros_like(ks)
    r = O.attend(q, Q._values(kc, ks, block), Q._values(vc, vs, block), [n], True, D ** -0.5)
    cache, _, _ = Q._cache(kc, vc, ks, vs, block)
    o, lse = torch.ones(1, M, 2, D, dtype=BF, device="cuda"), torch.zeros(1, 2, M, device="cuda")
    w = torch.zeros(1, 1, n, device="cuda") if weigh else None
    plan = ops.AttentionQ8Plan(q.cuda(), cache, o, kv_len=n, lse=lse, weight=w)
    if not weigh:
        plan.args.workspace, plan.args.workspace_bytes = None, 0     # one CTA sums all keys
    plan.run()
    Q._done()
    assert bool((o == 0).all())
    Q._check(o, lse, w, r, q, BF, D, [n], 2)


# ---------------------------------------------------------------------------------- probabilities in one part or in two

@pytest.mark.parametrize("single_p", [False, True])
@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("M,Hq,Hkv,D,S,block", [
    (1, 32, 2, 128, 16, 16),                     # a cluster for each unit
    (3, 16, 1, 64, 64, 32),
    (8, 16, 2, 128, 9100, 64),                   # pieces
    (40, 8, 2, 128, 16, 16),                     # tensor-core kernel
    (40, 8, 2, 64, 700, 64),                     # ... divided
])
def test_probabilities_are_two_parts_unless_one_is_asked_for(M, Hq, Hkv, D, S, block, dt, single_p):
    """Five positions of nearly equal weight whose values cancel in many columns: what the rounding of p leaves there is not
    hidden by the output's own rounding.  Queries are small, so that the scores' errors are."""
    n = 5
    q, kc, vc, ks, vs = Q._attend_inputs(1, M, Hq, Hkv, D, S, block, dt, 83)
    q = (q.float() * 2.0 ** -7).to(dt)
    vs[:] = 2.0 ** -6
    r = O.attend(q, Q._values(kc, ks, block), Q._values(vc, vs, block), [n], False, D ** -0.5)
    cache, _, _ = Q._cache(kc, vc, ks, vs, block)
    o = torch.zeros(1, M, Hq, D, dtype=dt, device="cuda")
    ops.attention_q8(q.cuda(), cache, o, kv_len=torch.tensor([n], dtype=torch.int32).cuda(), causal=False, single_p=single_p)
    Q._done()
    # as Q._tolerance, with the rounding of p that was asked for
    ds = (D + 8) * 2.0 ** -23 * r["T"].transpose(1, 2)[..., None] + 2.0 ** -21
    e = (o.double().cpu() - r["o"]).abs()
    near = lambda pe: torch.finfo(dt).eps / 2 * r["o"].abs() + (pe + 2 * ds) * r["A"] + 2.0 ** -25
    assert bool((e <= near(2.0 ** -11 if single_p else 2.0 ** -19)).all()), (e / near(2.0 ** -19)).max().item()
    if single_p:
        assert bool((e > near(2.0 ** -19)).any())          # one part it is


# ------------------------------------------------------------------------------------------------- queries and variants

@pytest.mark.parametrize("M,Hq,D,n,block,dt", [(6, 2, 64, 100, 16, HF), (40, 2, 128, 100, 16, BF), (40, 2, 64, 333, 32, HF), (200, 1, 128, 513, 32, BF),
                                               (200, 2, 64, 2100, 16, HF), (40, 3, 64, 140, 64, BF)])
def test_queries_that_are_not_finite_or_extreme(M, Hq, D, n, block, dt):
    """A row of q with an infinite or NaN element is NaN throughout and leaves its neighbours alone; tiny rows, rows of zeros, elements
    far below their row's largest: one head's rows 1 to 5, and rows near the end of a call of many."""
    q, kc, vc, ks, vs = Q._attend_inputs(1, M, Hq, 1, D, n, block, dt, 6)
    bad = torch.zeros(M, Hq, dtype=torch.bool)
    for r0 in {0, M - 6}:
        q[0, r0 + 1, 0, 3] = math.inf
        q[0, r0 + 2, Hq - 1, 7] = math.nan
        q[0, r0 + 3, 0] *= 2.0 ** (-120 if dt == BF else -20)
        q[0, r0 + 4, 0] = 0.0
        q[0, r0 + 5, Hq - 1, 0] = 2.0 ** (-60 if dt == BF else -22)
        bad[r0 + 1, 0] = bad[r0 + 2, Hq - 1] = True
    clean = torch.where(q.isfinite(), q, torch.zeros_like(q))
    r = O.attend(clean, Q._values(kc, ks, block), Q._values(vc, vs, block), [n], True, D ** -0.5)
    r["o"][0][bad] = math.nan
    r["lse"][0][bad.T] = math.nan
    cache, _, _ = Q._cache(kc, vc, ks, vs, block)
    o, lse = torch.zeros(1, M, Hq, D, dtype=dt, device="cuda"), torch.zeros(1, Hq, M, device="cuda")
    ops.attention_q8(q.cuda(), cache, o, kv_len=n, lse=lse)
    Q._done()
    Q._check(o, lse, None, r, clean, dt, D, [n], Hq)


VARIANTS = [
    # B, M, Hq, Hkv, D, S, lens, block, causal: one line for each form of the kernels
    (2, 2, 4, 1, 128, 300, [300, 77], 64, True),            # clusters: 8 rows, 16 rows, at head_dim 64 also 32
    (2, 4, 4, 1, 128, 300, [299, 3], 16, True),
    (2, 2, 4, 1, 64, 300, [300, 77], 64, True),
    (2, 4, 4, 1, 64, 300, [299, 3], 16, True),
    (2, 8, 4, 1, 64, 300, [299, 5], 32, True),
    (40, 1, 4, 4, 128, 1200, None, 32, True),               # shares, many units: two stages
    (2, 1, 4, 1, 128, 9100, [9100, 2], 128, True),          # few units: three
    (1, 3, 4, 1, 128, 9100, [9000], 16, True),
    (1, 2, 4, 1, 64, 9100, [9000], 16, True),
    (1, 3, 4, 1, 64, 9100, [9000], 16, True),
    (1, 8, 4, 1, 64, 9100, [9000], 16, True),
    (2, 40, 4, 2, 128, 300, [300, 41], 16, True),           # tensor-core kernel, scales of 16 and of 32 positions
    (2, 40, 4, 2, 128, 300, [300, 41], 32, True),
    (2, 40, 4, 2, 64, 300, [300, 41], 16, False),
    (2, 40, 4, 2, 64, 300, [300, 41], 128, True),
    (1, 40, 4, 2, 128, 2000, [1999], 16, True),             # ... divided
    (4, 257, 40, 8, 64, 5200, [0, 300, 257, 5200], 16, True),       # ... the last round in pieces
    (3, 257, 34, 17, 128, 5130, [5129, 258, 1], 32, True),
]


@pytest.mark.parametrize("single_p", [False, True])
@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("B,M,Hq,Hkv,D,S,lens,block,causal", VARIANTS)
def test_every_form_of_the_kernels(B, M, Hq, Hkv, D, S, lens, block, causal, dt, single_p):
    lens = [(i * 997) % (S + 1) for i in range(B)] if lens is None else lens
    q, kc, vc, ks, vs = Q._attend_inputs(B, M, Hq, Hkv, D, S, block, dt, 91)
    Q._spoil_behind(kc, vc, ks, vs, lens, block)
    o, lse, w, r = _call(q, kc, vc, ks, vs, lens, block, causal=causal, weigh=False, single_p=single_p)
    tol, ds = Q._tolerance(r, q, dt, D)
    if single_p:                                 # one part of p: off by 2^-11 of itself
        tol = tol + 2.0 ** -11 * r["A"]
    e = (o.double().cpu() - r["o"]).abs()
    assert bool((e <= tol).all()), (e / tol).max().item()
    far = r["lse"].isfinite()
    e = (lse.double().cpu() - r["lse"]).abs()
    assert torch.equal(lse.cpu() == -math.inf, ~far)
    assert bool((e <= ds[..., 0].transpose(1, 2) * 1.5 + 2.0 ** -21 * (1 + r["lse"].abs()))[far].all())


def test_the_largest_numbers_of_a_type_come_back_rounded():
    """fp16 up to 63487 and bf16 under 1.9375 * 2^127 stay finite through append and read; above, the nearest code is a power of two
    past the type's largest number."""
    for dt, below, above in ((HF, 63456.0, 63488.0), (BF, 1.9296875 * 2.0 ** 127, 1.9375 * 2.0 ** 127)):
        x = torch.zeros(1, 2, 1, 64, dtype=dt)
        x[0, 0], x[0, 1, 0, ::2] = below, above
        cache = ops.CacheQ8.empty(1, 16, 1, 64, block=16)
        out = torch.zeros(1, 2, 1, 64, dtype=dt, device="cuda")
        ops.cache_append(cache, x.cuda(), x.cuda(), kv_len=0)
        ops.cache_read(cache, out, out.clone(), kv_len=2)
        Q._done()
        assert bool(out[0, 0].isfinite().all()) and bool(out[0, 1, 0, ::2].isinf().all()) and bool((out[0, 1, 0, 1::2] == 0).all())


@pytest.mark.parametrize("M", [2, 16])
def test_weights_where_the_products_are_in_one_part(M):
    """Weights come from the scores: they do not depend on single_p."""
    q, kc, vc, ks, vs = Q._attend_inputs(1, M, 8, 2, 128, 2100, 32, BF, 97)
    ws = [_call(q, kc, vc, ks, vs, [2099], 32, weigh=True, single_p=sp)[2] for sp in (False, True)]
    assert torch.equal(*ws)
