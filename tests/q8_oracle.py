"""Plain 64-bit implementations of the 8-bit cache operators, for the tests (CPU tensors in, CPU tensors out)."""
import math

import torch

E4M3_MAX = 448.0


def e4m3_table() -> torch.Tensor:
    """Value of each of the 256 codes: sign, 4 exponent bits (bias 7), 3 mantissa bits, all ones NaN."""
    out = []
    for code in range(256):
        e, m = (code >> 3) & 15, code & 7
        v = math.ldexp(8 + m, e - 10) if e else math.ldexp(m, -9)
        out.append(math.nan if code & 127 == 127 else -v if code & 128 else v)
    return torch.tensor(out, dtype=torch.float64)


def decode(codes: torch.Tensor) -> torch.Tensor:
    return e4m3_table()[codes.view(torch.uint8).long()]


def to_grid(x: torch.Tensor) -> torch.Tensor:
    """Nearest e4m3 value, ties to the even mantissa."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3.0)
    return (torch.round(x / step) * step).clamp(-E4M3_MAX, E4M3_MAX)


def need_scale(x: torch.Tensor) -> float:
    """Smallest power of two 2^e, -64 <= e <= 120, with |x| <= 448 * 2^e over the finite elements."""
    fine = x[x.isfinite()].abs()
    amax = fine.max().item() if fine.numel() else 0.0
    e = -64
    while e < 120 and amax > E4M3_MAX * 2.0 ** e:
        e += 1
    return 2.0 ** e


def append(codes, scale, new, held, block):
    """codes [B, H, S, D] values (float64, the value each code stands for WITHOUT its scale), scale [B, H, nblk] float64, new [B, M, H, D],
    held [B]: returns (codes, scale) after the append."""
    codes, scale = codes.clone(), scale.clone()
    B, H, S, D = codes.shape
    M = new.shape[1]
    for b in range(B):
        n = int(held[b])
        for h in range(H):
            for j in range(n // block, (min(n + M, S) - 1) // block + 1):
                lo, hi = max(n, j * block), min(n + M, S, (j + 1) * block)
                if lo >= hi:
                    continue
                x = new[b, lo - n:hi - n, h].double()
                s = need_scale(x)
                if j * block < n:
                    old = scale[b, h, j].item()
                    if not old >= s:
                        codes[b, h, j * block:n] = to_grid(codes[b, h, j * block:n] * (old / s))
                    else:
                        s = old
                scale[b, h, j] = s
                codes[b, h, lo:hi] = torch.where(x.isfinite(), to_grid(x / s), torch.full_like(x, math.nan))
    return codes, scale


def attend(q, k, v, lens, causal, scale):
    """q [B, M, Hq, D], k / v [B, Hkv, S, D] float64 values.  Returns o [B, M, Hq, D], lse [B, Hq, M] (base 2), weight [B, Hkv, S],
    and two magnitudes the tolerances are made of: A [B, M, Hq, D] = sum p |v| and T [B, Hq, M] = max over visible positions
    of scale * sum |q k|."""
    B, M, Hq, D = q.shape
    Hkv, S = k.shape[1:3]
    G = Hq // Hkv
    q = q.double()
    o, A = torch.zeros(B, M, Hq, D, dtype=torch.float64), torch.zeros(B, M, Hq, D, dtype=torch.float64)
    lse, T = torch.full((B, Hq, M), -math.inf, dtype=torch.float64), torch.zeros(B, Hq, M, dtype=torch.float64)
    weight = torch.zeros(B, Hkv, S, dtype=torch.float64)
    for b in range(B):
        n = int(lens[b])
        if n == 0:
            continue
        see = torch.ones(M, n, dtype=torch.bool)
        if causal:
            see = torch.arange(n)[None, :] <= (n - M) + torch.arange(M)[:, None]
        some = see.any(1)
        for hq in range(Hq):
            h = hq // G
            kk, vv = k[b, h, :n], v[b, h, :n]
            x = (q[b, :, hq] @ kk.T * scale).masked_fill(~see, -math.inf)
            p = torch.where(some[:, None], torch.softmax(x, -1), torch.zeros_like(x)).masked_fill(~see, 0.0)
            bad = (see.double() @ vv.isnan().double()) > 0
            vz = vv.nan_to_num(0.0)
            o[b, :, hq] = (p @ vz).masked_fill(bad, math.nan)
            A[b, :, hq] = p @ vz.abs()
            T[b, hq] = (q[b, :, hq].abs() @ kk.abs().T * scale).masked_fill(~see, 0.0).amax(1)
            lse[b, hq] = torch.where(some, torch.logsumexp(x, -1) / math.log(2), torch.full_like(some, -math.inf, dtype=torch.float64))
            weight[b, h, :n] += p.sum(0)
    return dict(o=o, lse=lse, weight=weight, A=A, T=T)


def select(scores, n, keep, recent, first, G):
    """scores [Hs, n] -> kept positions per kv head [Hkv][m], and the group sums [Hkv, n] float32."""
    w = scores.double().reshape(scores.shape[0] // G, G, n).sum(1).float()
    out = []
    for row in w:
        if n <= keep:
            out.append(list(range(n)))
            continue
        always = [j for j in range(n) if j < first or j >= n - recent]
        # a NaN ranks above every number; equal scores by the lower position
        free = sorted((j for j in range(n) if not (j < first or j >= n - recent)),
                      key=lambda j: (not math.isnan(row[j]), -(row[j].item() if not math.isnan(row[j]) else 0.0), j))
        out.append(sorted(always + free[:keep - len(always)]))
    return out, w
