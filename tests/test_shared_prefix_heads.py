"""Attention of rows that share the first part of their cache with heads of every size that test_shared_prefix.py leaves out: layouts whose
loads lie across the halves of 16 keys (D % 32 != 0 in bfloat16), loads that the waves cannot share evenly, 32 keys a stage, one and two
waves a row.  Tolerances are those of test_shared_prefix.py.
"""
import pytest

from test_shared_prefix import BF16, F32, check, make, ops, plain, rows_behind, run, step_of

from mini_inference_engine_amd.kernels.shared_prefix import SharedPrefixPlan, _sharers
from mini_inference_engine_amd.kernels.variants import SHARED_HEAD_DIMS

SIZES = (112, 144, 160, 176, 192, 208, 224, 240)
# columns of one row alone, of several tiles with one that is not full, of more than a workgroup takes; keys that end inside a page and inside 32
CASES = [([(1, 0), (1, 0)], 70), ([(2, 33), (1, 0)], 40), ([(9, 130), (3, 64), (1, 5)], 100), ([(40, 333)], 20)]


def test_every_size_is_built_ahead():
    assert set(SIZES) < set(SHARED_HEAD_DIMS) and SHARED_HEAD_DIMS == tuple(range(16, 257, 16))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads", [(2, 2), (8, 1), (20, 1)])
@pytest.mark.parametrize("D", SIZES)
@pytest.mark.parametrize("case", range(len(CASES)))
def test_heads_of_other_sizes(ops, case, D, heads, dtype):
    groups, own = CASES[case]
    s = make(groups, rows_behind(groups, own, case), *heads, D, 16, dtype, seed=case)
    run(ops, s, groups, *heads, D, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("D", SIZES)
def test_items_of_a_wave_with_heads_of_other_sizes(ops, D, dtype):
    """Plans for one compute unit and for many, long pages, a row that sees nothing, a sink."""
    groups, Hq, Hkv = [(3, 200), (1, 0), (2, 31), (4, 0)], 6, 2
    positions = rows_behind(groups, 90, D)
    s = make(groups, positions, Hq, Hkv, D, 48, dtype, seed=D)
    contexts = [p + 1 for p in positions]
    s.positions[3] = -1
    step, group = step_of(s, most=max(contexts))
    want = plain(s, Hq, Hkv, D, D ** -0.5, 0.3)
    for units in (1, 600):
        for share in (True, False):
            plan = SharedPrefixPlan(groups, contexts, Hq, Hkv, D, "cuda", units=units, float32=dtype == F32, share=share)
            if units == 1:
                assert (plan.whole_items < plan.num_items) == (_sharers(D, dtype == F32) > 0)
            check(ops[dtype].shared_prefix_attention(s.q, Hq, Hkv, D, s.k, s.v, group, step, D ** -0.5, plan, sink=0.3), *want, D, dtype)
