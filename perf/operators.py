"""The operators of the 8-bit key/value cache, as a serving program calls them, beside their plain form.

Three operators that a decode loop runs one after the other:

  append  16-bit keys and values of M new tokens go into a cache of e4m3 codes with one scale for each block of
          `block` tokens and key/value head.  A scale is the smallest power of two 2^e with |x| <= 448 * 2^e for the
          block's new finite values, e within [-64, 120]; a block that already holds tokens keeps the larger of its
          scale and that one, and its older codes are rewritten where the scale grew.  What is not finite is held as
          NaN and does not count for the scale.  The result is read back as 16-bit values.
  attend  o = softmax(scale * q k^T) v over the first kv_len[b] cached tokens, query i of M seeing tokens up to
          kv_len[b] - M + i where causal; optionally each token's accumulated weight, summed over the queries and the
          query heads of its key/value head.
  evict   the `keep` tokens of each (sequence, key/value head) that stay: the first `first`, the last `recent`, and of the others
          those of the largest accumulated weight (summed over the score heads of a group, equal ones by the lower
          index); keys, values, scales and weights of these move to another cache in the order they had.

`own` chooses between the plain form (elementary torch operations in 32 bits) and the framework's kernels.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
E4M3_MAX = 448.0
SCALE_EXP_MIN, SCALE_EXP_MAX = -64, 120


# ---------------------------------------------------------------------------------------------------------- cases

def listed():
    llama, falcon = dict(Hq=32, Hkv=8, D=128), dict(Hq=71, Hkv=1, D=64)
    return [
        # one chat turn of one user: a single new token over about a thousand cached ones; latency is all that counts
        dict(name="decode, one sequence", kind="attend", dtype="bf16", B=1, M=1, block=32, lo=1040, hi=1040, S=1056,
             causal=True, weigh=False, **llama),
        # a speculative step or a short chunk, every query head with its own keys, weights kept for eviction
        dict(name="16 tokens, own keys, weights", kind="attend", dtype="fp16", B=1, M=16, Hq=32, Hkv=32, D=128,
             block=16, lo=1040, hi=1040, S=1040, causal=True, weigh=True),
        # a server's decode step: 32 users of different lengths, weights kept for eviction
        dict(name="decode, batch, weights", kind="attend", dtype="bf16", B=32, M=1, block=64, lo=1000, hi=8192, S=8192,
             causal=True, weigh=True, **llama),
        # decode over long documents
        dict(name="decode, long", kind="attend", dtype="fp16", B=2, M=1, block=128, lo=100001, hi=131071, S=131072,
             causal=True, weigh=False, **llama),
        # 71 query heads on one key/value head: few cached bytes, many rows for each
        dict(name="16 tokens, one shared head", kind="attend", dtype="bf16", B=4, M=16, block=16, lo=1040, hi=8189,
             S=8192, causal=True, weigh=False, **falcon),
        # a chunk of a long prompt: bound by the products
        dict(name="prompt chunk", kind="attend", dtype="bf16", B=2, M=2048, block=64, lo=8192, hi=8192, S=8192,
             causal=True, weigh=False, **llama),
        # one new token, one shared head
        dict(name="append, one token", kind="append", dtype="bf16", B=1, M=1, Hkv=1, D=64, block=16, lo=1039, hi=1039,
             S=1056),
        # chunks at odd places of caches of different lengths
        dict(name="append, chunks", kind="append", dtype="fp16", B=4, M=515, Hkv=8, D=128, block=32, lo=101, hi=1501,
             S=2048),
        # the prompts of a batch into empty caches
        dict(name="append, prompts", kind="append", dtype="bf16", B=8, M=2048, Hkv=8, D=128, block=64, lo=0, hi=0,
             S=2048),
        # half of a short 16-bit cache, one score for each head
        dict(name="evict, short, 16 bits", kind="evict", dtype="bf16", B=1, Hs=32, Hkv=32, D=128, block=0, lo=1040,
             hi=1040, S=1040, keep=520, recent=64, first=4, ties=True),
        # 1024 of 4096 tokens of an 8-bit cache, scores of 32 query heads for 8 key/value heads
        dict(name="evict, 8 bits", kind="evict", dtype="bf16", B=4, Hs=32, Hkv=8, D=128, block=64, lo=4096, hi=4096,
             S=4096, keep=1024, recent=256, first=4, ties=False),
        # long 16-bit caches with one shared head
        dict(name="evict, long, one shared head", kind="evict", dtype="fp16", B=2, Hs=71, Hkv=1, D=64, block=0,
             lo=30011, hi=32768, S=32768, keep=2048, recent=512, first=0, ties=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of the same ranges; never more work than the largest listed one of its kind."""
    kind = rng.choice(["attend", "attend", "append", "evict"])
    most = [work(c) for c in listed() if c["kind"] == kind]
    most_bytes, most_flops = max(w["bytes"] for w in most), max(w["flops"] for w in most)
    while True:
        Hq, Hkv, D = rng.choice([(32, 8, 128), (71, 1, 64), (32, 32, 128), (16, 2, 64), (40, 8, 128), (5, 1, 128)])
        c = dict(kind=kind, dtype=rng.choice(["bf16", "fp16"]), B=_log(rng, 1, 32), Hkv=Hkv, D=D,
                 block=rng.choice([16, 32, 64, 128]))
        if kind == "attend":
            decode = rng.random() < 0.6
            c.update(Hq=Hq, M=rng.choice([1, 1, 1, 2, 5, 8, 16]) if decode else _log(rng, 17, 2048),
                     causal=rng.random() < 0.85)
            c["weigh"] = decode and rng.random() < 0.4
            c["hi"] = c["M"] + _log(rng, 1, 131072) - 1
            c["lo"] = max(1, int(c["hi"] * rng.uniform(0.2, 1.0)))
            c["S"] = c["hi"] + rng.choice([0, 0, 1, 7, 100])
        elif kind == "append":
            c.update(M=1 if rng.random() < 0.3 else _log(rng, 1, 4096))
            c["hi"] = _log(rng, 1, 8192) - 1
            c["lo"] = int(c["hi"] * rng.uniform(0.0, 1.0))
            c["S"] = c["hi"] + c["M"] + rng.choice([0, 0, 1, 9, 130])
        else:
            c.update(Hs=rng.choice([Hkv, Hq]), hi=_log(rng, 2, 131072), ties=rng.random() < 0.5)
            c["block"] = rng.choice([0, 0, 16, 32, 64, 128])
            c["lo"] = max(1, int(c["hi"] * rng.uniform(0.3, 1.0)))
            c["S"] = c["hi"] + rng.choice([0, 0, 1, 33])
            c["keep"] = max(1, int(c["hi"] * rng.uniform(0.05, 0.9)))
            c["recent"] = int(c["keep"] * rng.choice([0.0, 0.1, 0.5]))
            c["first"] = min(rng.choice([0, 1, 4]), c["keep"] - c["recent"])
        w = work(c)
        if w["bytes"] <= most_bytes and w["flops"] <= most_flops and _state_bytes(c) <= 4e9:
            return c


def _lens(c):
    """Tokens in each sequence's cache: spread evenly from lo to hi."""
    n = max(1, c["B"] - 1)
    return [c["hi"]] if c["B"] == 1 else [c["lo"] + (c["hi"] - c["lo"]) * b // n for b in range(c["B"])]


def _state_bytes(c):
    return 2 * c["B"] * c["S"] * c["Hkv"] * c["D"] * (1 if c["block"] else 2) + 4 * c["B"] * c.get("Hs", 0) * c["S"]


def work(c):
    lens, B, Hkv, D = _lens(c), c["B"], c["Hkv"], c["D"]
    total = sum(lens)
    if c["kind"] == "attend":
        M, Hq = c["M"], c["Hq"]
        pairs = 0
        for n in lens:
            pairs += sum(max(0, n - M + i + 1) for i in range(M)) if c["causal"] else M * n
        scales = sum(-(-n // c["block"]) for n in lens) * Hkv * 8
        return {"bytes": 2 * 2 * B * M * Hq * D + 2 * total * Hkv * D + scales + (4 * total * Hkv if c["weigh"] else 0),
                "flops": 4 * Hq * D * pairs}
    if c["kind"] == "append":
        new, held = B * c["M"], total + B * c["M"]
        # new values and older codes in, the cache's 16-bit values and its scales out
        return {"bytes": Hkv * D * 2 * (2 * new + total + 2 * held) + 8 * Hkv * (held // c["block"] + B), "flops": 4 * new * Hkv * D}
    kept = sum(min(n, c["keep"]) for n in lens)
    # every score in, each kept row in and out, the indices and the kept scores out
    return {"bytes": 4 * total * c["Hs"] + 2 * kept * Hkv * D * (3 if c["block"] else 4) + 8 * kept * Hkv,
            "flops": total * c["Hs"]}


# --------------------------------------------------------------------------------------------------------- inputs

def _device():
    return torch.device("cuda" if torch.cuda.is_available() else "cpu")


def _rows(shape, dtype, g, spread=1.0):
    """Keys or values as projections give them: normal, some channels several times larger than the rest."""
    x = torch.randn(*shape, generator=g, device=g.device, dtype=torch.float32)
    channel = torch.rand(shape[1], 1, shape[-1], generator=g, device=g.device)
    return (x * (1.0 + 6.0 * (channel > 0.96)) * spread).to(dtype)


def _block_scales(x, block):
    """Power-of-two scale of each block of tokens of x [H, n, D] -> [H, blocks]."""
    H, n, D = x.shape
    blocks = -(-n // block)
    amax = torch.zeros(H, blocks * block, device=x.device)
    amax[:, :n] = x.float().abs().amax(-1)
    m, e = torch.frexp(amax.view(H, blocks, block).amax(-1) / E4M3_MAX)      # dividing by 7 * 2^6: judged exactly below
    e = torch.where(torch.ldexp(torch.full_like(m, E4M3_MAX), e - 1) >= amax.view(H, blocks, block).amax(-1), e - 1, e)
    return torch.ldexp(torch.ones_like(m), e.clamp(SCALE_EXP_MIN, SCALE_EXP_MAX))


def _fill(codes, scales, b, n, block, dtype, g, spread):
    """Sequence b's first n tokens hold rows in 8 bits; what lies behind them is left as it is."""
    H, D = codes.shape[1], codes.shape[3]
    for lo in range(0, n, 1 << 15):
        hi = min(n, lo + (1 << 15))
        x = _rows((1, H, hi - lo, D), dtype, g, spread)[0]
        s = _block_scales(x, block)
        codes[b, :, lo:hi] = (x.float() / s.repeat_interleave(block, 1)[:, :hi - lo, None]).to(torch.float8_e4m3fn).view(torch.uint8)
        scales[b, :, lo // block:lo // block + s.shape[1]] = s


def _cache(c, lens, g):
    """Codes and scales of a cache as earlier appends left it.  Rows behind a sequence's last hold what was there before: any byte."""
    B, Hkv, S, D, block = c["B"], c["Hkv"], c["S"], c["D"], c["block"]
    out = []
    for spread in (1.0, 0.5):
        codes = torch.randint(0, 256, (B, Hkv, S, D), generator=g, device=g.device, dtype=torch.uint8)
        scales = torch.full((B, Hkv, -(-S // block)), 1.0, device=g.device)
        for b, n in enumerate(lens):
            _fill(codes, scales, b, n, block, DTYPES[c["dtype"]], g, spread)
        out += [codes.view(torch.float8_e4m3fn), scales]
    return out


def prepare(c, seed):
    dev, dt = _device(), DTYPES[c["dtype"]]
    g = torch.Generator(device=dev).manual_seed(int(seed))
    lens, B, Hkv, D, S = _lens(c), c["B"], c["Hkv"], c["D"], c["S"]
    s = dict(case=c, lens=lens, kv_len=torch.tensor(lens, dtype=torch.int32, device=dev))
    if c["kind"] == "attend":
        s["k"], s["k_scale"], s["v"], s["v_scale"] = _cache(c, lens, g)
        s["q"] = torch.randn(B, c["M"], c["Hq"], D, generator=g, device=dev).to(dt)
        s["o"] = torch.zeros_like(s["q"])
        s["weight"] = torch.zeros(B, Hkv, S, device=dev) if c["weigh"] else None
    elif c["kind"] == "append":
        s["k"], s["k_scale"], s["v"], s["v_scale"] = _cache(c, lens, g)
        s["k_new"] = _rows((B, Hkv, c["M"], D), dt, g, 1.5).transpose(1, 2).contiguous()       # as a projection writes them
        s["v_new"] = _rows((B, Hkv, c["M"], D), dt, g, 0.75).transpose(1, 2).contiguous()
        s["k_out"], s["v_out"] = (torch.zeros(B, Hkv, S, D, device=dev, dtype=dt) for _ in range(2))
        s["held"] = s["kv_len"] + c["M"]
    else:
        if c["block"]:
            s["k"], s["k_scale"], s["v"], s["v_scale"] = _cache(c, lens, g)
        else:
            s["k"], s["v"] = (_rows((B, Hkv, S, D), dt, g) for _ in range(2))
        # accumulated softmax weights: positive, a few large, most small, the early tokens larger
        w = torch.exp(2.0 * torch.randn(B, c["Hs"], S, generator=g, device=dev))
        w = w / (1.0 + 0.01 * torch.arange(S, device=dev))
        s["scores"] = w.bfloat16().float() if c["ties"] else w              # statistics written in 16 bits are often equal
        keep = c["keep"]
        s["idx"] = torch.zeros(B, Hkv, keep, dtype=torch.int32, device=dev)
        s["kept_scores"] = torch.zeros(B, Hkv, keep, device=dev)
        s["kept_len"] = torch.zeros(B, dtype=torch.int32, device=dev)
        if c["block"]:
            s["k_to"], s["v_to"] = (torch.zeros(B, Hkv, keep, D, device=dev, dtype=torch.uint8).view(torch.float8_e4m3fn) for _ in range(2))
            s["ks_to"], s["vs_to"] = (torch.zeros(B, Hkv, -(-keep // c["block"]), device=dev) for _ in range(2))
        s["k_out"], s["v_out"] = (torch.zeros(B, Hkv, keep, D, device=dev, dtype=dt) for _ in range(2))
    if own:
        _plan(s)
    return s


def _plan(s):
    """What a program binds once for a cache and launches every step."""
    from triton_b200 import ops
    c = s["case"]
    if "k_scale" in s:
        cache = ops.CacheQ8(s["k"], s["v"], s["k_scale"], s["v_scale"], block=c["block"], layout="bhsd")
    if c["kind"] == "attend":
        s["plans"] = [ops.AttentionQ8Plan(s["q"], cache, s["o"], kv_len=s["kv_len"], causal=c["causal"],
                                          scale=c["D"] ** -0.5, weight=s["weight"])]
    elif c["kind"] == "append":
        s["plans"] = [ops.CacheAppendPlan(cache, s["k_new"], s["v_new"], kv_len=s["kv_len"]),
                      ops.CacheReadPlan(cache, ops.as_bshd(s["k_out"], "bhsd"), ops.as_bshd(s["v_out"], "bhsd"), kv_len=s["held"])]
    else:
        k_out, v_out = ops.as_bshd(s["k_out"], "bhsd"), ops.as_bshd(s["v_out"], "bhsd")
        if c["block"]:
            src, dst = cache, ops.CacheQ8(s["k_to"], s["v_to"], s["ks_to"], s["vs_to"], block=c["block"], layout="bhsd")
        else:
            src, dst = (ops.as_bshd(s["k"], "bhsd"), ops.as_bshd(s["v"], "bhsd")), (k_out, v_out)
        s["plans"] = [ops.CacheEvictPlan(src, dst, s["scores"], kv_len=s["kv_len"], keep=c["keep"], recent=c["recent"],
                                         first=c["first"], idx=s["idx"], scores_out=s["kept_scores"],
                                         kv_len_out=s["kept_len"])]
        if c["block"]:
            s["plans"].append(ops.CacheReadPlan(dst, k_out, v_out, kv_len=s["kept_len"]))


# ------------------------------------------------------------------------------------------------------------ run

def run(s):
    kind = s["case"]["kind"]
    if own:
        for p in s["plans"]:
            p.run()
    else:
        {"attend": _attend, "append": _append, "evict": _evict}[kind](s)
    if kind == "attend":
        return {"o": s["o"]} if s["weight"] is None else {"o": s["o"], "weight": s["weight"]}
    if kind == "append":
        return {"k": s["k_out"], "v": s["v_out"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    out = {"k": s["k_out"], "v": s["v_out"], "idx": s["idx"], "scores": s["kept_scores"], "len": s["kept_len"]}
    return dict(out, k_scale=s["ks_to"], v_scale=s["vs_to"]) if s["case"]["block"] else out


def _values(codes, scale, block, n):
    """The first n tokens' values of one sequence [H, S, D], in 32 bits."""
    return codes[:, :n].float() * scale.repeat_interleave(block, 1)[:, :n, None]


def _attend(s):
    c = s["case"]
    M, Hkv, D, T = c["M"], c["Hkv"], c["D"], c["block"]
    G = c["Hq"] // Hkv
    for b, n in enumerate(s["lens"]):
        k, v = _values(s["k"][b], s["k_scale"][b], T, n), _values(s["v"][b], s["v_scale"][b], T, n)
        q = s["q"][b].float().view(M, Hkv, G, D).permute(1, 2, 0, 3).reshape(Hkv, G * M, D)
        x = torch.bmm(q, k.transpose(1, 2)) * D ** -0.5                        # [Hkv, G * M, n]
        if c["causal"]:
            last = torch.arange(M, device=x.device).repeat(G) + (n - M)
            x = x.masked_fill(torch.arange(n, device=x.device)[None, :] > last[:, None], float("-inf"))
        top = x.amax(-1, keepdim=True).clamp_min(-3e38)                         # a row that sees nothing has weight nowhere
        p = torch.exp(x - top)
        total = p.sum(-1, keepdim=True)
        p = p / torch.where(total > 0, total, torch.ones_like(total))
        s["o"][b] = torch.bmm(p, v).view(Hkv, G, M, D).permute(2, 0, 1, 3).reshape(M, c["Hq"], D).to(s["o"].dtype)
        if s["weight"] is not None:
            s["weight"][b, :, :n] = p.sum(1)


def _append(s):
    c = s["case"]
    M, T, S = c["M"], c["block"], c["S"]
    for b, n in enumerate(s["lens"]):
        j0, j1 = n // T, (n + M - 1) // T + 1
        lo, hi = j0 * T, min(j1 * T, S)
        for codes, scale, new in ((s["k"], s["k_scale"], s["k_new"]), (s["v"], s["v_scale"], s["v_new"])):
            x = new[b].float().transpose(0, 1)                                  # [H, M, D]
            fine = torch.isfinite(x)
            amax = torch.zeros(x.shape[0], (j1 - j0) * T, device=x.device)
            amax[:, n - lo:n - lo + M] = torch.where(fine, x, torch.zeros_like(x)).abs().amax(-1)
            amax = amax.view(x.shape[0], j1 - j0, T).amax(-1)
            m, e = torch.frexp(amax)                                            # amax = m * 2^e, 448 = 0.875 * 2^9
            need = torch.ldexp(torch.ones_like(m), (e - 9 + (m > 0.875).int()).clamp(SCALE_EXP_MIN, SCALE_EXP_MAX))
            before = scale[b, :, j0:j1].clone()
            if n > lo:                                                          # the first block already holds tokens
                need[:, 0] = torch.maximum(need[:, 0], before[:, 0])
                held = codes[b, :, lo:n].float() * (before[:, 0] / need[:, 0])[:, None, None]
                codes[b, :, lo:n] = held.to(torch.float8_e4m3fn)
            scale[b, :, j0:j1] = need
            each = need.repeat_interleave(T, 1)[:, n - lo:n - lo + M, None]
            coded = torch.where(fine, x / each, torch.full_like(x, float("nan")))
            codes[b, :, n:n + M] = coded.to(torch.float8_e4m3fn)
        s["k_out"][b, :, :n + M] = _values(s["k"][b], s["k_scale"][b], T, n + M).to(s["k_out"].dtype)
        s["v_out"][b, :, :n + M] = _values(s["v"][b], s["v_scale"][b], T, n + M).to(s["v_out"].dtype)


def _evict(s):
    c = s["case"]
    Hkv, T, keep = c["Hkv"], c["block"], c["keep"]
    s["idx"].fill_(-1)
    s["kept_scores"].zero_()
    for b, n in enumerate(s["lens"]):
        w = s["scores"][b, :, :n].double().view(Hkv, -1, n).sum(1).float()      # 64 bits: what lies next to the border
        m = min(n, keep)
        rank = w.clone()
        rank[:, :c["first"]] = float("inf")
        rank[:, max(0, n - c["recent"]):] = float("inf")
        idx = torch.sort(rank, dim=-1, descending=True, stable=True).indices[:, :m].sort(-1).values
        s["idx"][b, :, :m] = idx.int()
        s["kept_scores"][b, :, :m] = torch.gather(w, 1, idx)
        s["kept_len"][b] = m
        at = idx[:, :, None].expand(-1, -1, c["D"])
        if not T:
            s["k_out"][b, :, :m] = torch.gather(s["k"][b], 1, at)
            s["v_out"][b, :, :m] = torch.gather(s["v"][b], 1, at)
            continue
        for codes, scale, to, scale_to, out in ((s["k"], s["k_scale"], s["k_to"], s["ks_to"], s["k_out"]),
                                                (s["v"], s["v_scale"], s["v_to"], s["vs_to"], s["v_out"])):
            each = torch.gather(scale[b], 1, idx // T)                          # [Hkv, m]: the scale each token had
            blocks = -(-m // T)
            wide = torch.zeros(Hkv, blocks * T, device=each.device)
            wide[:, :m] = each
            top = wide.view(Hkv, blocks, T).amax(-1)
            ratio = each / top.repeat_interleave(T, 1)[:, :m]
            held = torch.gather(codes[b].view(torch.uint8), 1, at).view(torch.float8_e4m3fn).float() * ratio[:, :, None]
            to[b, :, :m] = held.to(torch.float8_e4m3fn)
            scale_to[b, :, :blocks] = top
            out[b, :, :m] = _values(to[b], scale_to[b], T, m).to(out.dtype)


# ---------------------------------------------------------------------------------------------------------- exact

def _e4m3_table(dev):
    """The value of each of the 256 codes: sign, 4 exponent bits of bias 7, 3 mantissa bits; all ones is NaN."""
    out = []
    for code in range(256):
        e, m = (code >> 3) & 15, code & 7
        v = math.ldexp(8 + m, e - 10) if e else math.ldexp(m, -9)
        out.append(float("nan") if (code & 127) == 127 else -v if code & 128 else v)
    return torch.tensor(out, dtype=torch.float64, device=dev)


def _to_grid(x):
    """The e4m3 value nearest to each x, ties to the even mantissa (64 bits in and out)."""
    step = torch.exp2((torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6)))).clamp_min(-6.0) - 3.0)
    return (torch.round(x / step) * step).clamp(-E4M3_MAX, E4M3_MAX)


def _decoded(codes, scale, n, block):
    table = _e4m3_table(codes.device)
    at = torch.arange(n, device=codes.device) // block
    return table[codes.view(torch.uint8)[:, :n].long()] * scale.double()[:, at, None]


def exact(c, seed):
    """What run() returns, from the definition in 64 bits."""
    s = prepare(c, seed)
    return {"attend": _exact_attend, "append": _exact_append, "evict": _exact_evict}[c["kind"]](c, s)


def _exact_attend(c, s):
    M, Hkv, D, T, Hq = c["M"], c["Hkv"], c["D"], c["block"], c["Hq"]
    G = Hq // Hkv
    o = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    weight = torch.zeros(c["B"], Hkv, c["S"], dtype=torch.float64, device=o.device)
    for b, n in enumerate(s["lens"]):
        for h in range(Hkv):
            k = _decoded(s["k"][b, h:h + 1], s["k_scale"][b, h:h + 1], n, T)[0]
            v = _decoded(s["v"][b, h:h + 1], s["v_scale"][b, h:h + 1], n, T)[0]
            for i0 in range(0, M, 256):
                for g in range(G):
                    q = s["q"][b, i0:i0 + 256, h * G + g].double()
                    x = q @ k.T / math.sqrt(D)
                    if c["causal"]:
                        i = torch.arange(i0, i0 + q.shape[0], device=x.device)[:, None]
                        x[torch.arange(n, device=x.device)[None, :] - i > n - M] = -math.inf
                    p = torch.softmax(x, -1).nan_to_num(0.0)
                    o[b, i0:i0 + 256, h * G + g] = p @ v
                    weight[b, h, :n] += p.sum(0)
    return {"o": o, "weight": weight} if c["weigh"] else {"o": o}


def _exact_append(c, s):
    M, T, S = c["M"], c["block"], c["S"]
    out = {}
    for name in ("k", "v"):
        scale = s[name + "_scale"].double()
        values = torch.zeros(c["B"], c["Hkv"], S, c["D"], dtype=torch.float64, device=scale.device)
        for b, n in enumerate(s["lens"]):
            old, new = _decoded(s[name][b], s[name + "_scale"][b], n, T), s[name + "_new"][b].double().transpose(0, 1)
            row = values[b]
            row[:, :n] = old
            for j in range(n // T, (n + M - 1) // T + 1):
                lo, hi = max(n, j * T), min(n + M, (j + 1) * T)
                part = new[:, lo - n:hi - n]
                fine = part.isfinite()
                amax = torch.where(fine, part.abs(), torch.zeros_like(part)).flatten(1).amax(1)
                e = torch.ceil(torch.log2((amax / E4M3_MAX).clamp_min(2.0 ** SCALE_EXP_MIN))).clamp(SCALE_EXP_MIN, SCALE_EXP_MAX)
                need = torch.exp2(e)
                if j * T < n:
                    need = torch.maximum(need, scale[b, :, j])
                    row[:, j * T:n] = _to_grid(old[:, j * T:] / need[:, None, None]) * need[:, None, None]
                scale[b, :, j] = need
                coded = _to_grid(part / need[:, None, None]) * need[:, None, None]
                row[:, lo:hi] = torch.where(fine, coded, torch.full_like(coded, math.nan))
        out[name], out[name + "_scale"] = values, scale
    return out


def _exact_evict(c, s):
    Hkv, T, keep, B, D = c["Hkv"], c["block"], c["keep"], c["B"], c["D"]
    dev = s["scores"].device
    out = {"idx": torch.full((B, Hkv, keep), -1, dtype=torch.int32, device=dev),
           "scores": torch.zeros(B, Hkv, keep, dtype=torch.float64, device=dev),
           "len": torch.tensor([min(n, keep) for n in s["lens"]], dtype=torch.int32, device=dev)}
    for name in ("k", "v"):
        out[name] = torch.zeros(B, Hkv, keep, D, dtype=torch.float64, device=dev)
        if T:
            out[name + "_scale"] = torch.zeros(B, Hkv, -(-keep // T), dtype=torch.float64, device=dev)
    for b, n in enumerate(s["lens"]):
        m = min(n, keep)
        for h in range(Hkv):
            G = c["Hs"] // Hkv
            w = s["scores"][b, h * G:(h + 1) * G, :n].double().sum(0)
            # ordered by the weight as it is held, in 32 bits; argsort of the negated weights is stable
            order = torch.argsort(-w.float(), stable=True)
            free = order[(order >= c["first"]) & (order < n - c["recent"])]
            always = torch.tensor([j for j in range(n) if j < c["first"] or j >= n - c["recent"]], dtype=torch.long, device=dev)
            kept = torch.cat([always, free])[:m].sort().values if n > keep else torch.arange(n, device=dev)
            out["idx"][b, h, :m] = kept.int()
            out["scores"][b, h, :m] = w[kept]
            for name in ("k", "v"):
                if not T:
                    out[name][b, h, :m] = s[name][b, h, kept].double()
                    continue
                had = s[name + "_scale"][b, h].double()[kept // T]
                value = _e4m3_table(dev)[s[name][b, h].view(torch.uint8)[kept].long()] * had[:, None]
                top = torch.stack([part.max() for part in had.split(T)])
                out[name + "_scale"][b, h, :top.numel()] = top
                top = top[torch.arange(m, device=dev) // T, None]
                out[name][b, h, :m] = _to_grid(value / top) * top
    return out
