"""What the 8-bit cache operators refuse, judged before any CUDA call: no GPU needed (the pointers are never followed)."""
import ctypes as C

import pytest

from triton_b200 import _lib as L

NULL, SHAPE, ALIGN, DTYPE, VARIANT, WORKSPACE = -1, -2, -3, -4, -5, -6


@pytest.fixture(scope="module")
def lib():
    if not L.LIB_PATH.exists():
        from triton_b200.build import build
        build()
    return L.load()


def _ht(ptr, S, H, D):
    return L.TrnHeadTensor(ptr, S * H * D, D, S * D)


def _cache(base, S=256, H=2, D=64, block=32):
    nblk = -(-S // block) if block else 0
    sc = lambda p: L.TrnHeadTensor(p, nblk * H, 1, nblk)
    return L.TrnCacheQ8(_ht(base, S, H, D), _ht(base + (1 << 24), S, H, D), sc(base + (2 << 24)), sc(base + (3 << 24)), S, block)


def _append(**kw):
    a = L.TrnCacheAppendArgs(_cache(1 << 32), _ht(2 << 32, 3, 2, 64), _ht(3 << 32, 3, 2, 64), None, 5, 2, 3, 2, 64, L.TRN_BF16)
    return _with(a, kw)


def _read(**kw):
    a = L.TrnCacheReadArgs(_cache(1 << 32), _ht(2 << 32, 256, 2, 64), _ht(3 << 32, 256, 2, 64), 256, None, 5, 2, 2, 64, L.TRN_BF16)
    return _with(a, kw)


def _attend(**kw):
    a = L.TrnAttnQ8Args()
    a.q, a.o, a.cache = _ht(2 << 32, 3, 8, 64), _ht(3 << 32, 3, 8, 64), _cache(1 << 32)
    a.B, a.M, a.Hq, a.Hkv, a.D, a.dtype, a.scale, a.causal, a.kv_len_all = 2, 3, 8, 2, 64, L.TRN_BF16, 0.125, 1, 100
    return _with(a, kw)


def _evict(**kw):
    a = L.TrnCacheEvictArgs()
    a.src, a.dst, a.scores, a.idx = _cache(1 << 32), _cache(2 << 32), 3 << 32, 4 << 32
    a.score_stride_b, a.score_stride_h, a.Hs = 8 * 256, 256, 8
    a.B, a.Hkv, a.D, a.keep, a.recent, a.first, a.kv_len_all = 2, 2, 64, 100, 10, 2, 256
    return _with(a, kw)


def _with(a, kw):
    for path, value in kw.items():
        at, names = a, path.split("__")
        for n in names[:-1]:
            at = getattr(at, n)
        setattr(at, names[-1], value)
    return a


CACHE = [({"S": 0}, SHAPE), ({"S": -1}, SHAPE), ({"S": 1 << 30}, SHAPE), ({"block": 48}, SHAPE), ({"k__ptr": None}, NULL),
         ({"v__ptr": (1 << 32) + 8}, ALIGN), ({"k__stride_s": 72}, ALIGN), ({"k__stride_s": -64}, SHAPE), ({"v__stride_b": 0}, SHAPE),
         ({"k_scale__ptr": None}, NULL), ({"v_scale__ptr": (1 << 32) + 2}, ALIGN), ({"v_scale__stride_s": 0}, SHAPE)]


@pytest.mark.parametrize("change,code", CACHE)
@pytest.mark.parametrize("make,fn", [(_append, "trinity_cache_append"), (_read, "trinity_cache_read"), (_attend, "trinity_attention_q8")])
def test_caches_refused(lib, make, fn, change, code):
    assert getattr(lib, fn)(C.byref(make(**{"cache__" + k: v for k, v in change.items()})), None) == code


@pytest.mark.parametrize("make,fn,change,code", [
    (_append, "trinity_cache_append", dict(B=0), SHAPE),
    (_append, "trinity_cache_append", dict(M=0), SHAPE),
    (_append, "trinity_cache_append", dict(D=96), SHAPE),
    (_append, "trinity_cache_append", dict(dtype=7), DTYPE),
    (_append, "trinity_cache_append", dict(cache__block=0), SHAPE),
    (_append, "trinity_cache_append", dict(k_new__ptr=None), NULL),
    (_append, "trinity_cache_append", dict(v_new__stride_s=68), ALIGN),
    (_append, "trinity_cache_append", dict(v_new__stride_h=-64), SHAPE),
    (_read, "trinity_cache_read", dict(S_out=0), SHAPE),
    (_read, "trinity_cache_read", dict(k_out__ptr=None), NULL),
    (_read, "trinity_cache_read", dict(k_out__stride_s=0), SHAPE),
    (_read, "trinity_cache_read", dict(dtype=-1), DTYPE),
    (_attend, "trinity_attention_q8", dict(M=0), SHAPE),
    (_attend, "trinity_attention_q8", dict(Hq=9), SHAPE),
    (_attend, "trinity_attention_q8", dict(D=80), SHAPE),
    (_attend, "trinity_attention_q8", dict(scale=0.0), SHAPE),
    (_attend, "trinity_attention_q8", dict(scale=float("inf")), SHAPE),
    (_attend, "trinity_attention_q8", dict(scale=float("nan")), SHAPE),
    (_attend, "trinity_attention_q8", dict(dtype=2), DTYPE),
    (_attend, "trinity_attention_q8", dict(q__ptr=None), NULL),
    (_attend, "trinity_attention_q8", dict(o__ptr=(1 << 32) + 4), ALIGN),
    (_attend, "trinity_attention_q8", dict(o__stride_h=0), SHAPE),
    (_attend, "trinity_attention_q8", dict(weight=5 << 32, weight_stride_b=512, weight_stride_h=256, cache__S=100000, kv_len_all=100000), WORKSPACE),
    (_attend, "trinity_attention_q8", dict(weight=5 << 32, weight_stride_b=512, weight_stride_h=0), SHAPE),
    (_attend, "trinity_attention_q8", dict(weight=5 << 32, weight_stride_b=512, weight_stride_h=256, M=17), SHAPE),
    (_attend, "trinity_attention_q8", dict(workspace=(6 << 32) + 16, workspace_bytes=1 << 40, cache__S=100000, kv_len_all=100000), WORKSPACE),
    (_attend, "trinity_attention_q8", dict(workspace=6 << 32, workspace_bytes=100, cache__S=100000, kv_len_all=100000), WORKSPACE),
    (_evict, "trinity_cache_evict", dict(scores=None), NULL),
    (_evict, "trinity_cache_evict", dict(idx=None), NULL),
    (_evict, "trinity_cache_evict", dict(dst__block=64), VARIANT),
    (_evict, "trinity_cache_evict", dict(src__block=40, dst__block=40), SHAPE),
    (_evict, "trinity_cache_evict", dict(Hs=5), SHAPE),
    (_evict, "trinity_cache_evict", dict(Hs=0), SHAPE),
    (_evict, "trinity_cache_evict", dict(keep=0), SHAPE),
    (_evict, "trinity_cache_evict", dict(keep=257), SHAPE),                       # more than dst has room for
    (_evict, "trinity_cache_evict", dict(recent=99, first=2), SHAPE),
    (_evict, "trinity_cache_evict", dict(recent=-1), SHAPE),
    (_evict, "trinity_cache_evict", dict(first=2 ** 31 - 1, recent=2), SHAPE),
    (_evict, "trinity_cache_evict", dict(src__S=262145), SHAPE),
    (_evict, "trinity_cache_evict", dict(D=32), SHAPE),
    (_evict, "trinity_cache_evict", dict(score_stride_h=-1), SHAPE),
    (_evict, "trinity_cache_evict", dict(dst__k__ptr=1 << 32), VARIANT),          # dst over src
    (_evict, "trinity_cache_evict", dict(dst__v__ptr=(1 << 32) + 64 * 64), VARIANT),
    (_evict, "trinity_cache_evict", dict(dst__k_scale__ptr=(1 << 32) + (3 << 24)), VARIANT),
    (_evict, "trinity_cache_evict", dict(kv_len=7 << 32, kv_len_out=(7 << 32) + 4), VARIANT),
    (_evict, "trinity_cache_evict", dict(dst__v__stride_s=0), SHAPE),
    (_evict, "trinity_cache_evict", dict(src__k_scale__ptr=None), NULL),
])
def test_refused(lib, make, fn, change, code):
    assert getattr(lib, fn)(C.byref(make(**change)), None) == code


def test_null_argument_blocks(lib):
    for fn in ("trinity_cache_append", "trinity_cache_read", "trinity_attention_q8", "trinity_cache_evict"):
        assert getattr(lib, fn)(None, None) == NULL
    assert lib.trinity_attention_q8_workspace(None) == 0


def test_struct_layouts_match_the_header(tmp_path):
    import os
    import subprocess
    header = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "trinity_b200.h")
    structs = [L.TrnCacheQ8, L.TrnCacheAppendArgs, L.TrnCacheReadArgs, L.TrnAttnQ8Args, L.TrnCacheEvictArgs]
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{header}"', "int main(void) {"]
    for st in structs:
        lines.append(f'  printf("{st.__name__} %zu\\n", sizeof({st.__name__}));')
        lines += [f'  printf("{st.__name__}.{f} %zu\\n", offsetof({st.__name__}, {f}));' for f, _ in st._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["  return 0;", "}"]))
    subprocess.run(["gcc", "-std=c11", "-o", str(exe), str(src)], check=True)
    by = {st.__name__: st for st in structs}
    for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines():
        key, val = line.split()
        s, _, f = key.partition(".")
        assert (getattr(by[s], f).offset if f else C.sizeof(by[s])) == int(val), key


def test_python_refusals():
    import torch
    from triton_b200 import ops
    code = lambda *s: torch.zeros(*s, dtype=torch.uint8).view(torch.float8_e4m3fn)
    sc = torch.zeros(1, 2, 4)
    with pytest.raises(ValueError, match="16, 32, 64 or 128"):
        ops.CacheQ8(code(1, 2, 64, 64), code(1, 2, 64, 64), sc, sc, block=17)
    with pytest.raises(TypeError, match="float8_e4m3fn"):
        ops.CacheQ8(torch.zeros(1, 2, 64, 64), code(1, 2, 64, 64), sc, sc, block=16)
    with pytest.raises(ValueError, match="scales"):
        ops.CacheQ8(code(1, 2, 64, 64), code(1, 2, 64, 64), sc, sc, block=32)
    with pytest.raises(ValueError, match="same shape"):
        ops.CacheQ8(code(1, 2, 64, 64), code(1, 2, 32, 64), sc, sc, block=16)
    cache = ops.CacheQ8(code(1, 2, 64, 64), code(1, 2, 64, 64), sc, sc, block=16)
    row = torch.zeros(1, 3, 2, 64, dtype=torch.bfloat16)
    for n in (-1, 62):
        with pytest.raises(ValueError, match="does not fit"):
            ops.CacheAppendPlan(cache, row, row, kv_len=n)
    with pytest.raises(ValueError, match="int32"):
        ops.CacheAppendPlan(cache, row, row, kv_len=torch.zeros(1, dtype=torch.int64))
    with pytest.raises(ValueError, match="fit the cache"):
        ops.CacheAppendPlan(cache, row[..., :32], row[..., :32], kv_len=0)
    with pytest.raises(TypeError):
        ops.CacheAppendPlan(cache, row.float(), row.float(), kv_len=0)
    with pytest.raises(ValueError, match="no CPU path"):
        ops.CacheAppendPlan(cache, row, row, kv_len=0)
    q = torch.zeros(1, 3, 4, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="fit the cache"):
        ops.AttentionQ8Plan(q[:, :, :3], cache, q[:, :, :3].clone(), kv_len=3)
    with pytest.raises(ValueError, match="one shape and dtype"):
        ops.AttentionQ8Plan(q, cache, q.half(), kv_len=3)
    with pytest.raises(ValueError, match="weight"):
        ops.AttentionQ8Plan(q, cache, q.clone(), kv_len=3, weight=torch.zeros(1, 2, 63))
    many = torch.zeros(1, 17, 4, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="at most 16"):
        ops.AttentionQ8Plan(many, cache, many.clone(), kv_len=20, weight=torch.zeros(1, 2, 64))
    kv = (torch.zeros(1, 64, 2, 64, dtype=torch.bfloat16),) * 2
    s = torch.zeros(1, 2, 64)
    with pytest.raises(ValueError, match="one kind"):
        ops.CacheEvictPlan(cache, kv, s, kv_len=64, keep=8)
    with pytest.raises(ValueError, match="room for keep"):
        ops.CacheEvictPlan(kv, kv, s, kv_len=64, keep=65)
    with pytest.raises(ValueError, match="first \\+ recent"):
        ops.CacheEvictPlan(kv, kv, s, kv_len=64, keep=8, recent=8, first=1)
    with pytest.raises(ValueError, match="scores"):
        ops.CacheEvictPlan(kv, kv, s[:, :, :63], kv_len=64, keep=8)
    with pytest.raises(ValueError, match="scores"):
        ops.CacheEvictPlan(kv, kv, torch.zeros(1, 3, 64), kv_len=64, keep=8)
