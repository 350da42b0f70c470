"""The sizes that the GPU tests run reach every kernel form that the operators' range reaches."""
import ctypes

import pytest

from FlagOS_mhc import _C
from tests import sublayer_forms as SF


def spread(lo, hi, n):
    return sorted({round(lo * (hi / lo) ** (i / n)) for i in range(n + 1)})


def test_every_form_is_run():
    run = set().union(*(SF.linear_forms(*s) for s in SF.LINEAR_SHAPES),
                      *(SF.gated_forms(*s) for s in SF.GATED_SHAPES))
    reached = {}
    for T in spread(1, 65536, 24):
        for D in spread(64, 8192, 14):
            for F in spread(64, 16384, 16):
                for k in SF.linear_forms(T, D, F) | SF.gated_forms(T, D, F):
                    reached.setdefault(k, (T, D, F))
    assert len(reached) >= 150      # six products, three forms, their tiles and cuts
    assert not {k: s for k, s in reached.items() if k not in run}


@pytest.mark.parametrize("T,D,F", [(1, 64, 64), (48, 4096, 4096), (4096, 4096, 16384)])
def test_plan_query(T, D, F):
    for p in range(6):
        form, tile, cuts = SF.plan(p, T, D, F)
        assert cuts >= 1
        assert tile in {SF.STREAM: (8, 16), SF.CLUSTER: (32, 64, 128, 256), SF.PAIR: (256, 512)}[form]
    assert SF.plan(SF.GRAD_WEIGHT, T, D, F)[0] == SF.PAIR       # tokens are its summed dimension


def test_plan_query_refusals():
    o = [ctypes.byref(ctypes.c_int32()) for _ in range(3)]
    q = _C.lib().mhc_sublayer_plan
    for a in ((-1, 4, 4, 4), (6, 4, 4, 4), (0, 0, 4, 4), (0, -1, 4, 4), (0, 4, 0, 4), (0, 4, 4, 0)):
        assert q(*a, *o) == _C.MHC_ERR_INVALID_ARGUMENT
    for i in range(3):
        assert q(0, 4, 4, 4, *(None if j == i else v for j, v in enumerate(o))) == \
            _C.MHC_ERR_INVALID_ARGUMENT
