"""Sizes of the linear layer and the gated block that reach every kernel form of their matrix
products, and the query that says which.

A product takes one of three forms (``mhc_sublayer_plan``): weights streamed past a few tokens, a
cluster's tiles of 128 features by some tokens, or tiles of 256 or 512 rows on CTA pairs; the summed
dimension may be cut.  A form is run in depth where a tile's share of that dimension is longer than
the ring of stages that feeds it, and, on CTA pairs, in one round of tiles or in several.
"""
import ctypes

from FlagOS_mhc import _C

LINEAR, GRAD_X, GRAD_WEIGHT, GATE_UP, GATED_GRAD_HIDDEN, GATED_GRAD_X = range(6)
STREAM, CLUSTER, PAIR = range(3)
SMS = 148

# (T, D, F)
LINEAR_SHAPES = [
    (1, 64, 13416), (9, 64, 2999), (1, 4624, 688), (1, 4768, 1345), (1260, 64, 2472), (4994, 64, 713),
    (2431, 64, 1752), (593, 3728, 386), (260, 4744, 848), (40890, 64, 416), (4883, 64, 3928),
    (584, 398, 10896), (29223, 320, 299), (5244, 72, 8504), (9835, 64, 6735), (754, 6681, 1632),
    (668, 6200, 2360), (9752, 144, 9408), (12417, 144, 13240), (21619, 144, 10696),
    (12417, 13240, 144), (21619, 10696, 144)]
GATED_SHAPES = [
    (9, 88, 64), (1, 5280, 344), (17, 762, 9784), (34, 4944, 1000), (1339, 96, 1576), (246, 2560, 544),
    (10, 7984, 4360), (130, 424, 6648), (1879, 574, 397), (19112, 400, 64), (65, 3176, 2576),
    (934, 2552, 392), (6604, 536, 320), (1089, 4184, 264), (68, 5080, 5656), (628, 1880, 3176),
    (3027, 8064, 160), (6722, 64, 11331), (9728, 7105, 72), (4793, 5976, 232), (139, 6480, 10528),
    (279, 3120, 15032), (14608, 64, 14288), (19767, 144, 5312), (263, 6368, 12680),
    (10321, 8192, 64)]


def plan(product, T, D, F):
    """(form, tile, cuts)"""
    o = [ctypes.c_int32() for _ in range(3)]
    st = _C.lib().mhc_sublayer_plan(product, T, D, F, *map(ctypes.byref, o))
    assert st == _C.MHC_OK, st
    return tuple(v.value for v in o)


def _cdiv(a, b):
    return -(-a // b)


def forms(product, T, D, F):
    """What this product of these sizes runs: its form, and, where it runs it in depth, that too."""
    form, tile, cuts = plan(product, T, D, F)
    if form == STREAM:
        return {(product, form, tile)}
    # output rows and columns, and the summed dimension
    M, N, K = {LINEAR: (T, F, D), GRAD_X: (T, D, F), GRAD_WEIGHT: (F, D, T), GATE_UP: (T, F, D),
               GATED_GRAD_HIDDEN: (T, F, D), GATED_GRAD_X: (T, D, 2 * F)}[product]
    both = product == GATE_UP           # two weights side by side
    if form == CLUSTER:
        key = (product, form, tile, cuts)
        stages = min(10, (200 << 10) // ((2 if both else 1) * 16384 + tile * 128))
    else:
        units = _cdiv(M, tile) * _cdiv(N, 128 if both else 256) * cuts
        key = (product, form, tile, cuts > 1, "rounds" if units > SMS // 2 else "one")
        stages = 6 if tile == 256 else 4
    return {key, key + ("deep",)} if _cdiv(K, 64) // cuts > stages else {key}


def linear_forms(T, D, F):
    return set().union(*(forms(p, T, D, F) for p in (LINEAR, GRAD_X, GRAD_WEIGHT)))


def gated_forms(T, D, F):
    return set().union(forms(LINEAR, T, F, D), forms(GRAD_WEIGHT, T, F, D),
                       *(forms(p, T, D, F) for p in (GATE_UP, GATED_GRAD_HIDDEN, GATED_GRAD_X,
                                                     GRAD_WEIGHT)))
