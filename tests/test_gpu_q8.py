"""The 8-bit key/value cache on the GPU: append, read, attention and eviction against 64-bit oracles."""
import math

import pytest
import torch

import q8_oracle as O
from triton_b200 import _lib as L
from triton_b200 import ops

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def _codes(shape, g):
    """Random codes without NaN."""
    c = torch.randint(0, 256, shape, generator=g, dtype=torch.uint8)
    return torch.where((c & 127) == 127, c - 1, c)


def _layout(t, layout):
    """[B, H, S(, D)] -> the memory layout named."""
    return t.contiguous() if layout == "bhsd" else t.transpose(1, 2).contiguous()


def _scales(B, H, nblk, g, lo=-9, hi=-4):
    return torch.exp2(torch.randint(lo, hi, (B, H, nblk), generator=g).float())


def _cache(kc, vc, ks, vs, block, layout="bhsd"):
    dev = [_layout(t, layout).cuda().view(torch.float8_e4m3fn) for t in (kc, vc)]
    sc = [_layout(t, layout).cuda() for t in (ks, vs)]
    return ops.CacheQ8(*dev, *sc, block=block, layout=layout), dev, sc


def _values(codes, scale, block):
    return O.decode(codes) * scale.double().repeat_interleave(block, 2)[:, :, :codes.shape[2], None]


def _done():
    torch.cuda.synchronize()
    assert L.kernel_status() == 0


# ------------------------------------------------------------------------------------------------- append and read

APPEND = [
    # B, M, H, D, S, held, block, dtype, layout
    (1, 1, 1, 64, 16, [0], 16, BF, "bhsd"),
    (1, 1, 1, 64, 1, [0], 16, HF, "bhsd"),
    (3, 1, 2, 128, 50, [0, 15, 49], 16, BF, "bhsd"),
    (2, 5, 3, 64, 70, [62, 30], 32, HF, "bshd"),
    (2, 37, 2, 128, 200, [63, 64], 64, BF, "bshd"),
    (1, 300, 1, 128, 513, [129], 128, HF, "bhsd"),
    (2, 33, 2, 64, 100, [1, 95], 128, BF, "bhsd"),       # the second runs over the cache's end: dropped
    (1, 70, 1, 64, 40, [7], 16, BF, "bhsd"),             # more rows than the cache has room for
]


@pytest.mark.parametrize("B,M,H,D,S,held,block,dt,layout", APPEND)
def test_append_and_read(B, M, H, D, S, held, block, dt, layout):
    g = torch.Generator().manual_seed(7)
    nblk = -(-S // block)
    kc, vc = _codes((B, H, S, D), g), _codes((B, H, S, D), g)
    ks, vs = _scales(B, H, nblk, g), _scales(B, H, nblk, g, -3, 3)
    k = (torch.randn(B, M, H, D, generator=g) * torch.exp2(torch.randint(-6, 6, (B, M, 1, 1), generator=g).float())).to(dt)
    v = torch.randn(B, M, H, D, generator=g).to(dt)
    cache, dev, sc = _cache(kc, vc, ks, vs, block, layout)
    kv_len = torch.tensor(held, dtype=torch.int32).cuda()
    ops.cache_append(cache, k.cuda(), v.cuda(), kv_len=kv_len)
    _done()
    after = [min(n + M, S) for n in held]
    for i, (codes, scale, new) in enumerate(((kc, ks, k), (vc, vs, v))):
        want, want_s = O.append(O.decode(codes), scale.double(), new, held, block)
        got, got_s = cache.tensors()[i].cpu().transpose(1, 2), cache.tensors()[2 + i].cpu().transpose(1, 2)
        assert torch.equal(got_s.double(), want_s)
        for b in range(B):
            assert torch.equal(O.decode(got[b, :, :after[b]].contiguous()), want[b, :, :after[b]])
            # nothing behind the new rows is touched
            assert torch.equal(got[b, :, after[b]:].contiguous().view(torch.uint8), codes[b, :, after[b]:])
    # read back: the values, rounded once; what lies behind a sequence stays
    ko, vo = (torch.full((B, S, H, D), 7.0, dtype=dt, device="cuda") for _ in range(2))
    ops.cache_read(cache, ko, vo, kv_len=torch.tensor(after, dtype=torch.int32).cuda())
    _done()
    for i, out in enumerate((ko, vo)):
        val = (cache.tensors()[i].cpu().transpose(1, 2).float() *
               cache.tensors()[2 + i].cpu().transpose(1, 2).repeat_interleave(block, 2)[:, :, :S, None]).to(dt)
        for b in range(B):
            assert torch.equal(out[b, :after[b]].cpu(), val[b, :, :after[b]].transpose(0, 1))
            assert bool((out[b, after[b]:] == 7.0).all())


def test_append_token_by_token_equals_the_oracle_and_loses_nothing_above_the_smallest_code():
    """Scales grow while a block fills; codes are rewritten, exactly but for what falls under the smallest code."""
    g = torch.Generator().manual_seed(3)
    B, H, D, S, block = 1, 2, 64, 64, 32
    x = (torch.randn(B, S, H, D, generator=g) * torch.exp2(torch.arange(S).float() / 8)[None, :, None, None]).to(BF)
    cache = ops.CacheQ8.empty(B, S, H, D, block=block)
    kv_len = torch.zeros(B, dtype=torch.int32, device="cuda")
    row = x[:, :1].cuda()
    plan = ops.CacheAppendPlan(cache, row, row, kv_len=kv_len)
    codes, scale = torch.zeros(B, H, S, D, dtype=torch.float64), torch.zeros(B, H, S // block, dtype=torch.float64)
    for i in range(S):
        row.copy_(x[:, i:i + 1])
        plan.run()
        kv_len += 1
        codes, scale = O.append(codes, scale, x[:, i:i + 1], [i], block)
    _done()
    assert torch.equal(O.decode(cache.k.cpu().transpose(1, 2).contiguous()), codes)
    assert torch.equal(cache.v_scale.cpu().transpose(1, 2).double(), scale)
    # every element is within half a step of e4m3 (2^-4 of it, or half the smallest code) of what was appended: the
    # rewriting by powers of two adds a rounding only under the smallest normal code, 2^-6
    val = codes * scale.repeat_interleave(block, 2)[..., None]
    want = x.transpose(1, 2).double()
    small = scale.repeat_interleave(block, 2)[..., None] * 2.0 ** -9
    assert bool(((val - want).abs() <= torch.maximum(want.abs() * 2.0 ** -4, small)).all())


@pytest.mark.parametrize("dt", [BF, HF])
def test_append_of_what_is_not_finite_and_of_extremes(dt):
    x = torch.zeros(1, 16, 1, 64)
    x[0, 0, 0, :4] = torch.tensor([math.inf, -math.inf, math.nan, 1.0])
    x[0, 1, 0, 0] = 448.0 * 0.25                     # exactly at the border: scale 2^-2
    x[0, 2, 0, 0] = torch.finfo(dt).tiny
    x = x.to(dt)
    cache = ops.CacheQ8.empty(1, 32, 1, 64, block=16)
    ops.cache_append(cache, x.cuda(), (x * 0).nan_to_num(0.0).cuda(), kv_len=0)
    big = torch.full((1, 16, 1, 64), torch.finfo(dt).max, dtype=dt)
    ops.cache_append(cache, big.cuda(), big.cuda(), kv_len=16)
    _done()
    k = O.decode(cache.k.cpu()[0, :, 0])
    assert cache.k_scale.cpu()[0, 0, 0].item() == 0.25
    assert k[0, :3].isnan().all() and k[0, 3] == 4.0 and k[1, 0] == 448.0 and not k[1:16].isnan().any()
    assert cache.v_scale.cpu()[0, 0, 0].item() == 2.0 ** -64          # zeros
    s = cache.k_scale.cpu()[0, 1, 0].double()
    assert s == (2.0 ** 120 if dt == BF else 2.0 ** 8)                # 448 * 2^8 > 65504 > 448 * 2^7
    assert torch.equal(k[16:], O.to_grid(big[0, :, 0].double() / s))


def test_append_to_a_cache_with_foreign_scales():
    """A caller's own scales need not be powers of two: the larger one stays, new elements are divided by it."""
    g = torch.Generator().manual_seed(5)
    codes = _codes((1, 1, 32, 64), g)
    ks = torch.tensor([[[0.3, 0.7]]])
    x = torch.randn(1, 4, 1, 64, generator=g).to(BF)
    for factor in (1.0, 1e4):
        cache, _, _ = _cache(codes, codes, ks, ks, 16)
        y = (x * factor).to(BF)
        ops.cache_append(cache, y.cuda(), y.cuda(), kv_len=5)
        _done()
        got, s = O.decode(cache.k.cpu()[0, :, 0]), cache.k_scale.cpu()[0, :, 0].double()
        assert s[0] == (ks.double()[0, 0, 0] if factor == 1.0 else O.need_scale(y)) and s[1] == ks.double()[0, 0, 1]
        # half a step of e4m3 (2^-4 of the value, or 2^-10 under the smallest normal code) from the quotient as 32 bits hold it,
        # which is itself off by up to 2^-24 of the value: at a tie the two add up (0.3 * 3.75 / 128 is 2^-24 away from one)
        want = torch.cat([O.decode(codes)[0, 0, :5] * (ks[0, 0, 0].double() / s[0]), y[0, :, 0].double() / s[0]])
        half = torch.maximum(want.abs() * 2.0 ** -4, torch.full_like(want, 2.0 ** -10))
        assert bool(((got[:9] - want).abs() <= half + want.abs() * 2.0 ** -23).all())


# ------------------------------------------------------------------------------------------------------- attention

ATTEND = [
    # B, M, Hq, Hkv, D, S, lens, block, dtype, causal, layout
    (1, 1, 1, 1, 64, 1, [1], 16, BF, True, "bhsd"),
    (1, 1, 4, 1, 128, 33, [33], 16, HF, True, "bhsd"),
    (2, 1, 8, 2, 128, 200, [0, 131], 64, BF, True, "bhsd"),          # an empty sequence
    (3, 1, 8, 8, 64, 300, [1, 64, 299], 32, HF, True, "bshd"),
    (2, 4, 8, 2, 128, 500, [3, 477], 128, BF, True, "bhsd"),         # fewer positions than queries: a row sees nothing
    (2, 5, 10, 2, 64, 260, [260, 17], 16, HF, True, "bshd"),
    (1, 16, 4, 4, 128, 1040, [1040], 64, HF, True, "bhsd"),
    (1, 3, 71, 1, 64, 700, [613], 32, BF, True, "bhsd"),
    (2, 7, 4, 2, 64, 90, [90, 3], 16, BF, False, "bhsd"),            # not causal
    (1, 1, 32, 2, 128, 3000, [2977], 128, HF, True, "bhsd"),
    (2, 40, 6, 3, 128, 150, [150, 39], 32, BF, True, "bhsd"),
    (1, 130, 4, 2, 64, 300, [290], 64, HF, True, "bshd"),
    (1, 17, 20, 1, 128, 600, [600], 16, BF, False, "bhsd"),
    (2, 300, 4, 4, 128, 700, [700, 411], 128, BF, True, "bhsd"),
    (1, 257, 2, 1, 64, 257, [257], 16, HF, True, "bhsd"),
    (2, 64, 8, 1, 128, 2100, [2100, 1], 64, HF, True, "bshd"),
]


def _attend_inputs(B, M, Hq, Hkv, D, S, block, dt, seed, junk=None):
    g = torch.Generator().manual_seed(seed)
    kc, vc = _codes((B, Hkv, S, D), g), _codes((B, Hkv, S, D), g)
    # values of size ~1: codes are uniform over the format, so most are small and a few are hundreds
    kc = (torch.randn(B, Hkv, S, D, generator=g) * 40).to(torch.float8_e4m3fn).view(torch.uint8)
    nblk = -(-S // block)
    ks, vs = _scales(B, Hkv, nblk, g, -7, -4), _scales(B, Hkv, nblk, g, -9, 2)
    q = torch.randn(B, M, Hq, D, generator=g).to(dt)
    return q, kc, vc, ks, vs


def _spoil_behind(kc, vc, ks, vs, lens, block):
    """Behind a sequence's last position: NaN codes, and NaN or infinite scales in blocks that hold nothing."""
    for b, n in enumerate(lens):
        for t in (kc, vc):
            t[b, :, n:] = 0x7f
        for t in (ks, vs):
            t[b, :, -(-n // block):] = math.nan
            t[b, :, -(-n // block)::2] = math.inf


def _tolerance(r, q, dt, D):
    """Of o.  eps / 2 of the output for its rounding, and of A = sum p |v|: pe for the rounding of p in the product (one fp16:
    2^-11; two: below 2^-19), and 2 ds for the scores, whose absolute error ds (natural units) is below (D + 8) 2^-23 of T =
    scale * sum |q k| (a step of the fp32 accumulation each) and which enter the weights of the numerator and of the sum.  fp16: outputs below
    2^-14 have steps of 2^-24."""
    ds = (D + 8) * 2.0 ** -23 * r["T"].transpose(1, 2)[..., None] + 2.0 ** -21
    pe = 2.0 ** -11 if dt == BF else 2.0 ** -19
    return torch.finfo(dt).eps / 2 * r["o"].abs() + (pe + 2 * ds) * r["A"] + 2.0 ** -25, ds


def _check(o, lse, weight, r, q, dt, D, lens, G):
    tol, ds = _tolerance(r, q, dt, D)
    got = o.double().cpu()
    assert torch.equal(got.isnan(), r["o"].isnan())
    err = (got - r["o"]).abs()
    assert bool((err <= tol)[~r["o"].isnan()].all()), ((err / tol).nan_to_num(0).max().item(), err.nan_to_num(0).max().item())
    if lse is not None:
        got = lse.double().cpu()
        assert torch.equal(got == -math.inf, r["lse"] == -math.inf) and torch.equal(got.isnan(), r["lse"].isnan())
        e = (got - r["lse"]).abs()
        t = ds[..., 0].transpose(1, 2) * 1.5 + 2.0 ** -21 * (1 + r["lse"].abs())
        m = r["lse"].isfinite()
        assert bool((e <= t)[m].all())
    if weight is not None:
        # each row's p is off by at most 2 ds of itself, and the sum of R rows by R steps of 32 bits
        rel = 2 * ds.amax().item() + 2.0 ** -23 * q.shape[1] * G + 2.0 ** -20
        for b, n in enumerate(lens):
            e = (weight[b, :, :n].double().cpu() - r["weight"][b, :, :n]).abs()
            assert bool((e <= rel * r["weight"][b, :, :n] + 1e-30).all())


@pytest.mark.parametrize("B,M,Hq,Hkv,D,S,lens,block,dt,causal,layout", ATTEND)
def test_attention_q8(B, M, Hq, Hkv, D, S, lens, block, dt, causal, layout):
    q, kc, vc, ks, vs = _attend_inputs(B, M, Hq, Hkv, D, S, block, dt, 11)
    _spoil_behind(kc, vc, ks, vs, lens, block)
    scale = D ** -0.5
    r = O.attend(q, _values(kc, ks, block), _values(vc, vs, block), lens, causal, scale)
    cache, _, _ = _cache(kc, vc, ks, vs, block, layout)
    kv_len = torch.tensor(lens, dtype=torch.int32).cuda()
    weigh = M <= 16
    outs = []
    for rep in range(2):
        o = torch.full((B, M, Hq, D), 9.0, dtype=dt, device="cuda")
        lse = torch.full((B, Hq, M), 9.0, device="cuda")
        w = torch.full((B, Hkv, S + 3), 5.0, device="cuda") if weigh else None
        plan = ops.AttentionQ8Plan(q.cuda(), cache, o, kv_len=kv_len, causal=causal, lse=lse, weight=w)
        plan.run()
        _done()
        outs.append((o, lse, w))
    assert all(a is None or torch.equal(a.view(torch.int32) if a.dtype == torch.float32 else a.view(torch.int16),
                                        c.view(torch.int32) if c.dtype == torch.float32 else c.view(torch.int16))
               for a, c in zip(*outs))                                 # fixed order: bitwise the same
    _check(o, lse, w, r, q, dt, D, lens, Hq // Hkv)
    if weigh:
        for b, n in enumerate(lens):
            assert bool((w[b, :, n:] == 5.0).all())                    # behind the sequence: as it was
        # accumulation: one more call adds the same numbers
        before = w.clone()
        ops.attention_q8(q.cuda(), cache, o, kv_len=kv_len, causal=causal, weight=w, weight_add=True)
        _done()
        for b, n in enumerate(lens):
            assert bool(((w[b, :, :n] - 2 * before[b, :, :n]).abs() <= 2.0 ** -22 * w[b, :, :n]).all())
    # without scratch the key range is not divided: another order of sums, the same result within the tolerance
    if not weigh:
        a = ops.AttentionQ8Plan(q.cuda(), cache, o, kv_len=kv_len, causal=causal, lse=lse)
        a.args.workspace, a.args.workspace_bytes = None, 0
        o.fill_(9.0)
        a.run()
        _done()
        _check(o, lse, None, r, q, dt, D, lens, Hq // Hkv)


LONG = [
    # caches too long for one launch of clusters: shares of all chunks, pieces, the merge
    (3, 1, 8, 2, 128, 9100, [5000, 0, 9100], 64, BF, True),
    (2, 2, 6, 2, 64, 20000, [17, 19999], 16, HF, True),
    (40, 1, 4, 4, 64, 4500, None, 32, BF, True),                        # more units than CTAs, many lengths
    (1, 16, 2, 1, 128, 6000, [6000], 128, HF, True),                    # 32 rows: two tiles of 16
    (1, 3, 20, 1, 64, 7000, [6990], 16, BF, False),
    (1, 300, 2, 1, 64, 9000, [8999], 32, HF, True),                     # tensor-core kernel, keys divided among CTAs
    (2, 9, 71, 1, 64, 5000, [4990, 5], 16, BF, True),
    # more pairs of row tiles than SMs: 192 and 320, whole rounds and a rest in pieces
    (4, 257, 40, 8, 64, 5200, [0, 300, 257, 5200], 64, BF, True),
    (5, 130, 64, 32, 64, 700, [700, 699, 5, 0, 130], 16, HF, True),     # ... too short for pieces
]


@pytest.mark.parametrize("workspace", [True, False])
@pytest.mark.parametrize("B,M,Hq,Hkv,D,S,lens,block,dt,causal", LONG)
def test_attention_q8_long(B, M, Hq, Hkv, D, S, lens, block, dt, causal, workspace):
    lens = [(i * 997) % (S + 1) for i in range(B)] if lens is None else lens
    q, kc, vc, ks, vs = _attend_inputs(B, M, Hq, Hkv, D, S, block, dt, 41)
    _spoil_behind(kc, vc, ks, vs, lens, block)
    r = O.attend(q, _values(kc, ks, block), _values(vc, vs, block), lens, causal, D ** -0.5)
    cache, _, _ = _cache(kc, vc, ks, vs, block)
    o = torch.full((B, M, Hq, D), 9.0, dtype=dt, device="cuda")
    lse = torch.full((B, Hq, M), 9.0, device="cuda")
    w = torch.full((B, Hkv, S + 1), 5.0, device="cuda") if workspace and M <= 16 else None
    plan = ops.AttentionQ8Plan(q.cuda(), cache, o, kv_len=torch.tensor(lens, dtype=torch.int32).cuda(), causal=causal, lse=lse, weight=w)
    if not workspace:
        plan.args.workspace, plan.args.workspace_bytes = None, 0         # the key range is not divided
    plan.run()
    _done()
    _check(o, lse, w, r, q, dt, D, lens, Hq // Hkv)
    first = o.clone()
    if w is not None:
        assert all(bool((w[b, :, n:] == 5.0).all()) for b, n in enumerate(lens))
    plan.run()
    _done()
    assert torch.equal(o, first)


@pytest.mark.parametrize("B,M,Hq,Hkv,D,S,lens,block,dt,causal", [
    # weights with the rows of a kv head shared by a CTA's threads: 128 positions or 32 a CTA
    (5, 10, 32, 8, 64, 603, [603, 1, 0, 9, 129], 32, BF, True),         # 40 rows, more CTAs than SMs
    (5, 10, 32, 8, 128, 601, [601, 128, 127, 11, 33], 16, HF, False),
    (1, 11, 6, 2, 128, 130, [129], 64, BF, True),                       # 33 rows, few CTAs
    (3, 16, 16, 1, 64, 290, [290, 31, 15], 16, HF, True),               # 256 rows
    (2, 15, 17, 1, 64, 97, [97, 3], 16, BF, True),                      # 255 rows
    (1, 16, 512, 1, 64, 70, [69], 32, BF, True),                        # 8192 rows, the most there may be
])
def test_weights_of_many_rows(B, M, Hq, Hkv, D, S, lens, block, dt, causal):
    q, kc, vc, ks, vs = _attend_inputs(B, M, Hq, Hkv, D, S, block, dt, 47)
    _spoil_behind(kc, vc, ks, vs, lens, block)
    r = O.attend(q, _values(kc, ks, block), _values(vc, vs, block), lens, causal, D ** -0.5)
    cache, _, _ = _cache(kc, vc, ks, vs, block)
    o = torch.full((B, M, Hq, D), 9.0, dtype=dt, device="cuda")
    lse = torch.full((B, Hq, M), 9.0, device="cuda")
    w = torch.full((B, Hkv, S + 1), 5.0, device="cuda")
    plan = ops.AttentionQ8Plan(q.cuda(), cache, o, kv_len=torch.tensor(lens, dtype=torch.int32).cuda(), causal=causal, lse=lse, weight=w)
    plan.run()
    _done()
    _check(o, lse, w, r, q, dt, D, lens, Hq // Hkv)
    assert all(bool((w[b, :, n:] == 5.0).all()) for b, n in enumerate(lens))
    first = w.clone()
    plan.run()
    _done()
    assert torch.equal(w, first)


def test_lengths_outside_the_cache_count_as_the_nearer_end():
    B, Hq, Hkv, D, S, block, dt = 2, 4, 2, 64, 60, 16, BF
    q, kc, vc, ks, vs = _attend_inputs(B, 1, Hq, Hkv, D, S, block, dt, 43)
    cache, _, _ = _cache(kc, vc, ks, vs, block)
    want = ops.attention_q8(q.cuda(), cache, kv_len=torch.tensor([0, S], dtype=torch.int32).cuda())
    got = ops.attention_q8(q.cuda(), cache, kv_len=torch.tensor([-3, S + 9], dtype=torch.int32).cuda())
    before = [t.clone() for t in cache.tensors()[2:]] + [t.view(torch.uint8).clone() for t in cache.tensors()[:2]]
    k = torch.randn(B, 3, Hkv, D, device="cuda").to(dt)
    ops.cache_append(cache, k, k, kv_len=torch.full((B,), S + 1, dtype=torch.int32, device="cuda"))      # nothing fits
    out = torch.zeros(B, S, Hkv, D, dtype=dt, device="cuda")
    ops.cache_read(cache, out[:, :50], out[:, :50].clone(), kv_len=torch.tensor([-1, S + 1], dtype=torch.int32).cuda())
    _done()
    assert torch.equal(want, got)
    after = [t for t in cache.tensors()[2:]] + [t.view(torch.uint8) for t in cache.tensors()[:2]]
    assert all(torch.equal(a, c) for a, c in zip(before, after))
    assert bool((out[0] == 0).all()) and bool((out[1, 50:] == 0).all()) and bool((out[1, :50] != 0).any())


@pytest.mark.parametrize("which", ["position", "batch"])
def test_offsets_beyond_32_bits(which):
    """Caches spread over gigabytes: strides of positions or of batch items that carry offsets past 2^32 bytes."""
    B, S, Hkv, D, block = 2, 150, 1, 64, 16
    g = torch.Generator().manual_seed(47)
    wide = 9_000_000_000
    sb, ss = (D, 32_000_000) if which == "position" else (4_400_000_000, D)
    buf = torch.zeros(wide, dtype=torch.uint8, device="cuda")
    cache = ops.CacheQ8.empty(B, S, Hkv, D, block=block, layout="bshd")
    spread = [buf[o:].as_strided((B, S, Hkv, D), (sb, ss, D, 1)).view(torch.float8_e4m3fn) for o in (0, 4 * D * S)]
    far = ops.CacheQ8(*spread, torch.zeros(B, -(-S // block), Hkv, device="cuda"), torch.zeros(B, -(-S // block), Hkv, device="cuda"),
                      block=block, layout="bshd")
    k, v = torch.randn(B, S, Hkv, D, generator=g).to(BF).cuda(), torch.randn(B, S, Hkv, D, generator=g).to(BF).cuda()
    outs = []
    for c in (cache, far):
        ops.cache_append(c, k, v, kv_len=0)
        ko, vo = torch.zeros_like(k), torch.zeros_like(v)
        ops.cache_read(c, ko, vo, kv_len=S)
        small = ops.attention_q8(k[:, :4].contiguous(), c, kv_len=S)
        large = ops.attention_q8(k[:, :100].contiguous(), c, kv_len=S)
        to = ops.CacheQ8.empty(B, 40, Hkv, D, block=block, layout="bshd")
        idx = ops.cache_evict(c, to, torch.rand(B, 1, S, generator=torch.Generator().manual_seed(1)).cuda(), kv_len=S, keep=40)
        outs.append((ko, vo, small, large, idx, to.k.view(torch.uint8), to.v_scale))
    _done()
    assert all(torch.equal(a, c) for a, c in zip(*outs))


@pytest.mark.parametrize("M,Hq,Hkv,D,n,block,dt", [(4, 4, 2, 128, 77, 16, BF), (8, 4, 1, 64, 200, 32, HF), (160, 2, 1, 128, 300, 64, BF),
                                                   (40, 8, 2, 64, 170, 16, HF)])
def test_attention_q8_nan_reaches_exactly_the_rows_that_see_it(M, Hq, Hkv, D, n, block, dt):
    """NaN codes among the newest positions: rows that do not see them stay as they are, rows that do are NaN (k: all of the
    row; v: that column)."""
    q, kc, vc, ks, vs = _attend_inputs(1, M, Hq, Hkv, D, n, block, dt, 5)
    vc[0, 0, n - M // 2, 3] = 0x7f
    vc[0, 0, n - 1, D - 1] = 0xff
    vc[0, Hkv - 1, n - M, 0] = 0x7f                  # seen by all but no earlier row
    kc[0, Hkv - 1, n - 2, 5] = 0xff
    r = O.attend(q, _values(kc, ks, block), _values(vc, vs, block), [n], True, D ** -0.5)
    assert r["o"].isnan().any() and not r["o"][0, 0].isnan().all()
    cache, _, _ = _cache(kc, vc, ks, vs, block)
    o, lse = torch.zeros(1, M, Hq, D, dtype=dt, device="cuda"), torch.zeros(1, Hq, M, device="cuda")
    ops.attention_q8(q.cuda(), cache, o, kv_len=n, lse=lse)
    _done()
    _check(o, lse, None, r, q, dt, D, [n], Hq // Hkv)


def test_attention_q8_rows_of_q_that_are_not_finite_or_extreme():
    dt, D, n = BF, 128, 100
    q, kc, vc, ks, vs = _attend_inputs(1, 6, 2, 1, D, n, 32, dt, 6)
    q[0, 1, 0, 3] = math.inf
    q[0, 2, 1, 7] = math.nan
    q[0, 3, 0] *= 2.0 ** -120                        # the whole row tiny: uniform weights
    q[0, 4, 0] = 0.0
    q[0, 5, 1, 0] = 2.0 ** -60                       # far below the row's largest
    cache, _, _ = _cache(kc, vc, ks, vs, 32)
    o, lse = torch.zeros(1, 6, 2, D, dtype=dt, device="cuda"), torch.zeros(1, 2, 6, device="cuda")
    ops.attention_q8(q.cuda(), cache, o, kv_len=n, lse=lse)
    _done()
    bad = torch.zeros(6, 2, dtype=torch.bool)
    bad[1, 0] = bad[2, 1] = True
    assert torch.equal(o.isnan().any(-1)[0].cpu(), bad) and torch.equal(o.isnan().all(-1)[0].cpu(), bad)
    qf = q.clone()
    qf[0, 1, 0, 3] = qf[0, 2, 1, 7] = 0.0
    r = O.attend(qf, _values(kc, ks, 32), _values(vc, vs, 32), [n], True, D ** -0.5)
    r["o"][0][bad] = math.nan
    r["lse"][0][bad.T] = math.nan
    _check(o, lse, None, r, qf, dt, D, [n], 2)


def test_attention_q8_scales_far_apart_and_zero():
    """Blocks whose value scales are 2^40 apart, and a block of zeros whose scale is 0."""
    dt, D, n, block = HF, 64, 150, 16
    q, kc, vc, ks, vs = _attend_inputs(1, 2, 4, 2, D, n, block, dt, 8)
    vs[0, :, 1] = 2.0 ** -40
    vs[0, :, 3] = 0.0
    vs[0, :, 5] = 2.0 ** -64
    ks[0, :, 2] = 0.0
    r = O.attend(q, _values(kc, ks, block), _values(vc, vs, block), [n], True, D ** -0.5)
    cache, _, _ = _cache(kc, vc, ks, vs, block)
    o, lse = torch.zeros(1, 2, 4, D, dtype=dt, device="cuda"), torch.zeros(1, 4, 2, device="cuda")
    w = torch.zeros(1, 2, n, device="cuda")
    ops.attention_q8(q.cuda(), cache, o, kv_len=n, lse=lse, weight=w)
    _done()
    _check(o, lse, w, r, q, dt, D, [n], 2)


def test_attention_q8_strided_queries_and_outputs():
    """q as a slice of a wider projection, o head-major, a cache that is a slice of a larger one."""
    dt, B, M, Hq, Hkv, D, S, n, block = BF, 2, 3, 4, 2, 64, 80, 75, 16
    q, kc, vc, ks, vs = _attend_inputs(B, M, Hq, Hkv, D, S, block, dt, 9)
    r = O.attend(q, _values(kc, ks, block), _values(vc, vs, block), [n, n], True, D ** -0.5)
    wide = torch.zeros(B, M, Hq + 3, D, dtype=dt, device="cuda")
    wide[:, :, 2:2 + Hq] = q.cuda()
    both = torch.zeros(B, S, 2, Hkv, D, dtype=torch.uint8, device="cuda")           # keys and values interleaved
    both[:, :, 0], both[:, :, 1] = kc.cuda().transpose(1, 2), vc.cuda().transpose(1, 2)
    both = both.view(torch.float8_e4m3fn)
    cache = ops.CacheQ8(both[:, :, 0], both[:, :, 1], ks.cuda().transpose(1, 2), vs.cuda().transpose(1, 2), block=block, layout="bshd")
    o = torch.zeros(B, Hq, M, D, dtype=dt, device="cuda")
    ops.attention_q8(wide[:, :, 2:2 + Hq], cache, ops.as_bshd(o, "bhsd"), kv_len=n)
    _done()
    _check(o.transpose(1, 2), None, None, r, q, dt, D, [n, n], 2)


# -------------------------------------------------------------------------------------------------------- eviction

EVICT = [
    # B, Hs, Hkv, D, S, lens, keep, recent, first, block (0: 16 bits), dtype, layout
    (1, 1, 1, 64, 1, [1], 1, 0, 0, 0, BF, "bhsd"),
    (2, 4, 2, 128, 100, [100, 0], 30, 5, 2, 0, BF, "bhsd"),
    (2, 2, 2, 64, 77, [77, 20], 33, 33, 0, 16, HF, "bshd"),           # nothing but recent ones
    (1, 6, 3, 128, 1500, [1499], 700, 100, 4, 32, BF, "bhsd"),
    (3, 2, 1, 64, 5000, [5000, 1024, 3], 129, 0, 0, 0, HF, "bshd"),
    (1, 1, 1, 128, 40000, [39999], 2000, 64, 4, 128, BF, "bhsd"),
    (2, 71, 1, 64, 3000, [3000, 2999], 1024, 1, 1, 64, BF, "bhsd"),
    (1, 2, 2, 64, 300, [300], 300, 10, 0, 16, HF, "bhsd"),            # everything stays
]


def _check_evict(src_codes, scale, dst, dst_scale, kept, block, b, h, pad):
    """One (b, h) of an 8-bit cache against the definition; pad: what the destination held before."""
    m = len(kept)
    val = O.decode(src_codes[b, h])[kept]
    s = scale[b, h].double()[torch.tensor(kept, dtype=torch.long) // block] if m else torch.zeros(0)
    for j in range(0, m, block):
        top = s[j:j + block].max()
        assert dst_scale[b, h, j // block].double() == top
        want = O.to_grid(val[j:j + block] * (s[j:j + block] / top)[:, None])
        got = O.decode(dst[b, h, j:min(j + block, m)].contiguous())
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(0.0), want.nan_to_num(0.0))
    assert bool((dst[b, h, m:].view(torch.uint8) == pad).all())


@pytest.mark.parametrize("kind", ["plain", "ties", "odd"])
@pytest.mark.parametrize("B,Hs,Hkv,D,S,lens,keep,recent,first,block,dt,layout", EVICT)
def test_evict(B, Hs, Hkv, D, S, lens, keep, recent, first, block, dt, layout, kind):
    g = torch.Generator().manual_seed(13)
    scores = torch.rand(B, Hs, S, generator=g)
    if kind == "ties":
        scores = (scores * 4).floor()                                  # four values: the border lies among equals
    if kind == "odd":
        scores = torch.randn(B, Hs, S, generator=g) * 1e20             # negative ones, zeros of both signs, infinities, NaN
        at = torch.randint(0, S, (B, Hs, max(1, S // 5)), generator=g)
        scores.scatter_(2, at, torch.tensor([0.0, -0.0, math.inf, 1e-42, math.nan])[torch.randint(0, 5, at.shape, generator=g)])
        if Hs > Hkv:
            scores = scores.nan_to_num(0.0, posinf=0.0)                # sums of infinities are tested where there are none to add
    for b, n in enumerate(lens):
        scores[b, :, n:] = math.inf                                    # behind the sequence: never chosen
    kv_len = torch.tensor(lens, dtype=torch.int32).cuda()
    idx = torch.full((B, Hkv, keep), 99, dtype=torch.int32, device="cuda")
    sout, lout = torch.full((B, Hkv, keep), 99.0, device="cuda"), torch.zeros(B, dtype=torch.int32, device="cuda")
    kw = dict(kv_len=kv_len, keep=keep, recent=recent, first=first, idx=idx, scores_out=sout, kv_len_out=lout)
    if block:
        nblk = -(-S // block)
        kc, vc = _codes((B, Hkv, S, D), g), _codes((B, Hkv, S, D), g)
        kc[:, :, ::7, 1] = 0x7f                                        # NaN codes move as they are
        ks, vs = _scales(B, Hkv, nblk, g), _scales(B, Hkv, nblk, g)
        cache, _, _ = _cache(kc, vc, ks, vs, block, layout)
        dst = ops.CacheQ8.empty(B, keep + 5, Hkv, D, block=block, layout=layout)
        ops.cache_evict(cache, dst, scores.cuda(), **kw)
    else:
        kc, vc = torch.randn(B, Hkv, S, D, generator=g).to(dt), torch.randn(B, Hkv, S, D, generator=g).to(dt)
        k, v = (ops.as_bshd(_layout(t, layout).cuda(), layout) for t in (kc, vc))
        dk, dv = (torch.full((B, Hkv, keep + 5, D), 3.0, dtype=dt, device="cuda") for _ in range(2))
        ops.cache_evict((k, v), (ops.as_bshd(dk, "bhsd"), ops.as_bshd(dv, "bhsd")), scores.cuda(), **kw)
    _done()
    for b, n in enumerate(lens):
        kept, w = O.select(scores[b, :, :n], n, keep, recent, first, Hs // Hkv)
        assert lout[b].item() == min(n, keep)
        for h in range(Hkv):
            m = len(kept[h])
            assert idx[b, h].tolist() == kept[h] + [-1] * (keep - m)
            assert torch.equal(sout[b, h, :m].cpu().nan_to_num(-7.0), w[h][kept[h]].nan_to_num(-7.0)) and bool((sout[b, h, m:] == 0).all())
            if block:
                for codes, scale, to, to_s in ((kc, ks, dst.k, dst.k_scale), (vc, vs, dst.v, dst.v_scale)):
                    _check_evict(codes, scale, to.cpu().transpose(1, 2), to_s.cpu().transpose(1, 2), kept[h], block, b, h, 0)
            else:
                for have, to in ((kc, dk), (vc, dv)):
                    assert torch.equal(to[b, h, :m].cpu(), have[b, h][kept[h]]) and bool((to[b, h, m:] == 3.0).all())


def test_evict_sums_the_same_with_and_without_scratch():
    B, Hs, Hkv, n, keep = 2, 21, 3, 9001, 1000
    g = torch.Generator().manual_seed(51)
    scores = torch.exp(3 * torch.randn(B, Hs, n, generator=g))
    k = torch.randn(B, n, Hkv, 64, generator=g).to(BF).cuda()
    kv_len = torch.tensor([n, 5000], dtype=torch.int32).cuda()
    outs = []
    for scratch in (True, False):
        to, sout = torch.zeros(B, keep, Hkv, 64, dtype=BF, device="cuda"), torch.zeros(B, Hkv, keep, device="cuda")
        plan = ops.CacheEvictPlan((k, k), (to, to.clone()), scores.cuda(), kv_len=kv_len, keep=keep, recent=7, first=2, scores_out=sout)
        assert plan.args.workspace_bytes == 4 * B * Hkv * n
        if not scratch:
            plan.args.workspace = None
        plan.run()
        _done()
        outs.append((plan.idx, sout, to))
    assert all(torch.equal(a, c) for a, c in zip(*outs))
    for b, m in enumerate((n, 5000)):
        kept, w = O.select(scores[b, :, :m], m, keep, 7, 2, Hs // Hkv)
        for h in range(Hkv):
            assert outs[0][0][b, h].tolist() == kept[h] and torch.equal(outs[0][1][b, h].cpu(), w[h][kept[h]])


def test_evict_long_rows_with_many_equals():
    """262144 positions, the longest a call takes, three values only."""
    S, keep = 262144, 70001
    g = torch.Generator().manual_seed(2)
    scores = torch.randint(0, 3, (1, 1, S), generator=g).float()
    k = torch.arange(S, device="cuda", dtype=torch.int32).view(1, S, 1, 1).expand(1, S, 1, 32).contiguous().view(HF)
    to = torch.zeros(1, keep, 1, 64, dtype=HF, device="cuda")
    to2 = torch.zeros_like(to)
    idx = ops.cache_evict((k, k), (to, to2), scores.cuda(), kv_len=S, keep=keep, recent=100, first=3)
    _done()
    w = scores[0, 0].clone()
    w[:3] = 9
    w[-100:] = 9
    want = torch.sort(w, descending=True, stable=True).indices[:keep].sort().values
    assert torch.equal(idx[0, 0].cpu().long(), want)
    assert torch.equal(to.view(torch.int32)[0, :, 0, 0].cpu().long(), want) and torch.equal(to.view(torch.int32), to2.view(torch.int32))


# --------------------------------------------------------------------------------------- together, streams, graphs

def test_a_decode_loop_with_eviction():
    """Prompt -> decode steps that append, attend and accumulate weights -> eviction -> more steps, against the oracle
    carried along in 64 bits (fed with the codes the device holds, so that every step is judged by itself)."""
    B, Hq, Hkv, D, block, S, keep = 2, 8, 2, 64, 16, 96, 40
    dt, g = BF, torch.Generator().manual_seed(17)
    lens = [50, 33]
    kv_len = torch.zeros(B, dtype=torch.int32, device="cuda")
    caches = [ops.CacheQ8.empty(B, S, Hkv, D, block=block) for _ in range(2)]
    prompt = [torch.randn(B, 50, Hkv, D, generator=g).to(dt) for _ in range(2)]
    ops.cache_append(caches[0], prompt[0].cuda(), prompt[1].cuda(), kv_len=kv_len)
    kv_len.copy_(torch.tensor(lens))                 # the second prompt is shorter: its padding is behind its last position
    acc = torch.zeros(B, Hkv, S, device="cuda")
    want = torch.zeros(B, Hkv, S, dtype=torch.float64)
    now = 0
    for step in range(30):
        if step == 14:
            idx = torch.zeros(B, Hkv, keep, dtype=torch.int32, device="cuda")
            kept, left = torch.zeros(B, Hkv, keep, device="cuda"), torch.zeros(B, dtype=torch.int32, device="cuda")
            ops.cache_evict(caches[0], caches[1], acc, kv_len=kv_len, keep=keep, recent=8, first=2, idx=idx, scores_out=kept, kv_len_out=left)
            _done()
            for b in range(B):
                sel, _ = O.select(acc[b, :, :lens[b]].cpu(), lens[b], keep, 8, 2, 1)
                assert idx[b].tolist() == [s + [-1] * (keep - len(s)) for s in sel]
            acc.zero_()
            acc[:, :, :keep] = kept
            want = acc.double().cpu()
            kv_len.copy_(left)
            lens = left.tolist()
            now = 1
        cache = caches[now]
        q, k, v = (torch.randn(B, 1, h, D, generator=g).to(dt) for h in (Hq, Hkv, Hkv))
        ops.cache_append(cache, k.cuda(), v.cuda(), kv_len=kv_len)
        kv_len += 1
        lens = [n + 1 for n in lens]
        o = ops.attention_q8(q.cuda(), cache, kv_len=kv_len, weight=acc, weight_add=True)
        _done()
        kc, vc = (t.cpu().transpose(1, 2).contiguous() for t in (cache.k, cache.v))
        ks, vs = (t.cpu().transpose(1, 2).contiguous() for t in (cache.k_scale, cache.v_scale))
        # what was appended is held to half a step of e4m3
        for b, n in enumerate(lens):
            new = _values(kc, ks, block)[b, :, n - 1]
            assert bool(((new - k[b, 0].double()).abs() <= torch.maximum(k[b, 0].double().abs() * 2.0 ** -4,
                                                                         ks[b, :, (n - 1) // block, None].double() * 2.0 ** -10)).all())
        r = O.attend(q, _values(kc, ks, block), _values(vc, vs, block), lens, True, D ** -0.5)
        _check(o, None, None, r, q, dt, D, lens, Hq // Hkv)
        for b, n in enumerate(lens):
            want[b, :, :n] += r["weight"][b, :, :n]
            assert bool(((acc[b, :, :n].double().cpu() - want[b, :, :n]).abs() <= 1e-3 * want[b, :, :n]).all())


@pytest.mark.parametrize("S", [600, 9000])            # one launch of clusters; shares and the merge
def test_captured_steps_replay_with_growing_lengths(S):
    """append + lengths + attention captured once; replays equal direct calls bit for bit.  Two graphs that share one scratch
    area, replayed one after the other."""
    B, Hq, Hkv, D, block, dt = 2, 8, 2, 128, 32, HF
    g = torch.Generator().manual_seed(23)
    def fresh():
        gg = torch.Generator().manual_seed(29)
        q, kc, vc, ks, vs = _attend_inputs(B, 1, Hq, Hkv, D, S, block, dt, 29)
        cache, _, _ = _cache(kc, vc, ks, vs, block)
        return dict(cache=cache, q=q.cuda(), k=torch.randn(B, 1, Hkv, D, generator=gg).to(dt).cuda(), o=torch.zeros(B, 1, Hq, D, dtype=dt, device="cuda"),
                    n=torch.tensor([S - 100, 37], dtype=torch.int32, device="cuda"), w=torch.zeros(B, Hkv, S, device="cuda"))
    ws = torch.empty(ops.attention_q8_workspace_bytes(B, 1, Hq, Hkv, D, S, weight=True), dtype=torch.uint8, device="cuda")
    def step(t):
        t["append"].run()
        t["n"] += 1
        t["attend"].run()
    def bind(t):
        t["append"] = ops.CacheAppendPlan(t["cache"], t["k"], t["k"], kv_len=t["n"])
        t["attend"] = ops.AttentionQ8Plan(t["q"], t["cache"], t["o"], kv_len=t["n"], weight=t["w"], weight_add=True, workspace=ws)
    direct, graphs = fresh(), [fresh(), fresh()]
    for t in [direct] + graphs:
        bind(t)
    for _ in range(5):
        step(direct)
    _done()
    side = torch.cuda.Stream()
    captured = []
    for t in graphs:
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(t)                                    # warm-up on the capturing stream: this is the first step
        torch.cuda.current_stream().wait_stream(side)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            step(t)
        captured.append(gr)
    for _ in range(4):
        for gr in captured:
            gr.replay()
    _done()
    for t in graphs:
        assert torch.equal(t["n"], direct["n"]) and torch.equal(t["o"], direct["o"]) and torch.equal(t["w"], direct["w"])
        assert torch.equal(t["cache"].k.view(torch.uint8), direct["cache"].k.view(torch.uint8))


@pytest.mark.parametrize("M,S", [(1, 300), (1, 9000), (40, 3000)])
def test_plain_stream_order_equals_dependent_launch(M, S, monkeypatch):
    """TRINITY_NO_PDL=1 (plain launches) gives the same bits, on the way through append, attention and eviction."""
    B, Hq, Hkv, D, block, dt, keep = 2, 8, 2, 64, 32, BF, 100
    outs = []
    for plain in (False, True):
        if plain:
            monkeypatch.setenv("TRINITY_NO_PDL", "1")
        q, kc, vc, ks, vs = _attend_inputs(B, M, Hq, Hkv, D, S, block, dt, 61)
        cache, _, _ = _cache(kc, vc, ks, vs, block)
        to = ops.CacheQ8.empty(B, keep, Hkv, D, block=block)
        rows = q[:, :, :Hkv].contiguous().cuda()
        w = torch.rand(B, Hkv, S, generator=torch.Generator().manual_seed(1)).cuda()
        ops.cache_append(cache, rows, rows, kv_len=S - M)
        o = ops.attention_q8(q.cuda(), cache, kv_len=S, **(dict(weight=w, weight_add=True) if M <= 16 else {}))
        idx = ops.cache_evict(cache, to, w, kv_len=S, keep=keep, recent=5)
        k16, v16 = (torch.zeros(B, keep, Hkv, D, dtype=dt, device="cuda") for _ in range(2))
        ops.cache_read(to, k16, v16, kv_len=keep)
        _done()
        outs.append((o, idx, w, k16, v16))
    assert all(torch.equal(a, c) for a, c in zip(*outs))


def test_two_streams_at_once():
    """The same call on two streams, each with its own plan: the results of one stream alone."""
    B, M, Hq, Hkv, D, S, block, dt = 1, 2, 8, 2, 64, 2000, 64, BF
    q, kc, vc, ks, vs = _attend_inputs(B, M, Hq, Hkv, D, S, block, dt, 31)
    cache, _, _ = _cache(kc, vc, ks, vs, block)
    qd = q.cuda()
    alone = ops.attention_q8(qd, cache, kv_len=S)
    outs = [torch.zeros_like(alone) for _ in range(2)]
    plans = [ops.AttentionQ8Plan(qd, cache, o, kv_len=S) for o in outs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, p in zip(streams, plans):
            with torch.cuda.stream(s):
                p.run()
    _done()
    assert all(torch.equal(o, alone) for o in outs)
