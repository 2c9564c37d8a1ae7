"""What eviction refuses beside what test_q8_refusals.py holds: no GPU needed."""
import ctypes as C

import pytest

import test_q8_refusals as R
from test_q8_refusals import lib  # noqa: F401  (fixture)

# scores of _evict: 2 items x 8 heads x 256 positions of 4 bytes from 3 << 32; idx: 2 x 2 x 100 from 4 << 32
SCORES, END = 3 << 32, (3 << 32) + 2 * 8 * 256 * 4


@pytest.mark.parametrize("change", [
    dict(scores_out=SCORES),                                       # compaction in place
    dict(scores_out=END - 4),
    dict(scores_out=SCORES - 2 * 2 * 100 * 4 + 4),
    dict(idx=SCORES + 4096),
    dict(kv_len_out=SCORES + 8),
    dict(idx=7 << 32, kv_len=(7 << 32) + 16),
    dict(scores_out=(4 << 32) + 400),                              # over idx
    dict(scores_out=5 << 32, kv_len_out=(5 << 32) + 4),
    dict(Hs=258, score_stride_b=258 * 256, workspace=SCORES + 256, workspace_bytes=1 << 30),
    dict(Hs=258, score_stride_b=258 * 256, workspace=(4 << 32) - 256, workspace_bytes=1 << 30),
])
def test_results_over_what_is_read_or_over_one_another(lib, change):  # noqa: F811
    assert lib.trinity_cache_evict(C.byref(R._evict(**change)), None) == R.VARIANT


@pytest.mark.parametrize("change", [
    dict(scores_out=END, kv_len=5 << 32, kv_len_out=6 << 32),      # side by side
    dict(idx=SCORES - 2 * 2 * 100 * 4),
    dict(kv_len=7 << 32, kv_len_out=(7 << 32) + 8),
    dict(scores_out=(4 << 32) + 1600),
    dict(workspace=SCORES + 256, workspace_bytes=1 << 30),         # this shape uses none
])
def test_neighbours_are_not_refused(lib, change):  # noqa: F811
    """Judged as fit: what answers then is the missing GPU."""
    import torch
    if torch.cuda.is_available():
        pytest.skip("the pointers are not memory")
    assert lib.trinity_cache_evict(C.byref(R._evict(**change)), None) in (-7, -8)


@pytest.mark.parametrize("keep", [2 ** 29 + 1, 2 ** 31 - 1000, 2 ** 31 - 1])
def test_more_rows_to_keep_than_32_bit_steps_reach(lib, keep):  # noqa: F811
    """A destination with room for 2^31 rows: the loop that marks the unused ones steps past the largest int."""
    assert lib.trinity_cache_evict(C.byref(R._evict(keep=keep, dst__S=keep, dst__k__stride_b=2 ** 40, dst__v__stride_b=2 ** 40, dst__k__stride_h=2 ** 38,
                                                    dst__v__stride_h=2 ** 38, dst__k__ptr=1 << 48, dst__v__ptr=1 << 49, dst__k_scale__ptr=1 << 50,
                                                    dst__v_scale__ptr=1 << 51, idx=1 << 52)), None) == R.SHAPE
