"""Which kernel the products of a language model's layers take on a full MI355X (256 compute units), checked on the host.  The
tables name, for every form, a product that takes it; the GPU tests run these (test_grouped_forms_gpu.py, test_xent_forms_gpu.py,
test_w4_precision_gpu.py), so a form that a later choice gives to other sizes is missed here and not silently left out there."""
import ctypes

import numpy as np
import pytest

import t2sp_amd

CODES = {"float32": 0, "float16": 1, "bfloat16": 2}
BOTH, ALL = ["float16", "bfloat16"], ["float32", "float16", "bfloat16"]


def ragged(T, E, seed=0):
    """T rows in E groups: a large one, empty ones, the rest anyhow."""
    rng = np.random.default_rng(seed)
    share = rng.random(E) ** 2 + 0.02
    if E > 2:
        share[rng.integers(0, E)] = 0
        share[E // 2] = share.sum() * 0.7
    return [int(n) for n in rng.multinomial(T, share / share.sum())]


# (straight from memory, rows of a tile), types, opb, rows of the groups, K, N
FORWARD = [
    ((True, 16), ["float32"], 0, [5, 0, 3], 72, 72), ((True, 16), ["float32"], 1, [8, 0], 72, 72),
    ((True, 16), BOTH, 0, [7, 0, 1], 520, 72), ((True, 16), BOTH, 1, [7, 0, 1], 72, 72),
    ((True, 32), ["float32"], 0, ragged(410, 16), 1032, 520), ((True, 32), ["float32"], 1, ragged(1500, 40), 72, 72),
    ((True, 32), BOTH, 0, ragged(1000, 40), 1032, 264), ((True, 32), BOTH, 1, ragged(1000, 40), 1032, 264),
    ((True, 64), ["float32"], 0, ragged(100, 24), 1032, 72), ((True, 64), ["float32"], 1, [130], 264, 2056),
    ((True, 64), BOTH, 0, ragged(100, 24), 2056, 72), ((True, 64), BOTH, 1, [130], 1032, 2056),
    ((False, 64), ["float32"], 0, ragged(3000, 8), 72, 72), ((False, 64), ["float32"], 1, ragged(1500, 4), 72, 136),
    ((False, 64), BOTH, 0, [60, 40], 72, 72), ((False, 64), BOTH, 1, ragged(2100, 6), 72, 72),
    ((False, 128), ["float32"], 0, [700, 300], 72, 2056), ((False, 128), ["float32"], 1, ragged(1000, 4), 72, 2056),
    ((False, 128), BOTH, 0, ragged(6000, 16), 72, 264), ((False, 128), BOTH, 1, ragged(4100, 4), 72, 520),
    ((False, 256), BOTH, 0, ragged(8200, 16), 264, 1032), ((False, 256), BOTH, 1, ragged(8200, 16), 264, 1032),
    ((False, 256), BOTH, 0, [1000, 100, 257, 643], 520, 4104), ((False, 256), BOTH, 1, [1000, 100, 257, 643], 520, 4104),
]
# tile, whether the rows are summed in parts, types, rows of the groups, K, N
WGRAD = [
    (128, False, ALL, [90, 0, 46], 264, 520), (128, True, ALL, [2400, 600], 264, 520),
    (256, False, BOTH, ragged(1300, 20), 520, 520), (256, False, BOTH, [1500, 0, 700, 800], 1032, 2056),
]
# the logits' tile (forward), the gradient's (logits, dH, its parts > 1, dW, its parts > 1), types, T, V, D
XENT = [
    (64, (64, 128, True, 128, False), ALL, 100, 300, 64), (128, (128, 128, True, 128, True), ["float32"], 300, 10001, 64),
    (128, (128, 128, True, 128, False), BOTH, 100, 20001, 264), (256, (256, 256, True, 256, False), BOTH, 200, 50001, 136),
    (256, (256, 256, True, 256, False), BOTH, 1500, 20001, 520), (64, (64, 128, True, 256, False), BOTH, 100, 10001, 1032),
    (64, (64, 256, False, 128, True), BOTH, 777, 300, 1032), (64, (64, 128, False, 128, True), ["float32"], 4100, 300, 1032),
]
# tiles of x, of the matrix, types, M, N, K, group
W4 = [
    (1, 4, ALL, 1, 16397, 296, 128), (1, 4, BOTH, 9, 16397, 296, 32), (1, 4, BOTH, 16, 16397, 296, 64), (2, 2, BOTH, 20, 8205, 296, 64),
    (4, 2, BOTH, 50, 8205, 296, 32), (4, 2, BOTH, 70, 8205, 296, 128), (2, 1, ALL, 20, 100, 296, 64), (4, 1, ALL, 50, 100, 296, 64),
    (2, 1, ALL, 50, 100, 290, 64), (1, 1, ["float32"], 9, 16397, 296, 32),
]


@pytest.fixture
def lib():
    L = t2sp_amd.lib()
    L.t2sp_set_machine.argtypes = [ctypes.c_int, ctypes.c_int]
    L.t2sp_set_machine.restype = None
    L.t2sp_set_machine(256, 8)
    yield L
    L.t2sp_set_machine(0, 0)


def forward_form(L, dtype, opb, T, E, K, N):
    few = ctypes.c_int(-1)
    rows = L.t2sp_gemm_grouped_plan(CODES[dtype], opb, T, E, K, N, ctypes.byref(few))
    return bool(few.value), rows


def wgrad_form(L, dtype, T, E, K, N):
    parts = ctypes.c_int(-1)
    tile = L.t2sp_gemm_grouped_wgrad_plan(CODES[dtype], T, E, K, N, ctypes.byref(parts))
    return tile, parts.value > 1


def xent_form(L, dtype, T, V, D, rounded=0):
    out = (ctypes.c_int * 5)()
    piece = L.t2sp_xent_grad_plan(CODES[dtype], rounded, T, V, D, out)
    return L.t2sp_xent_plan(CODES[dtype], T, V, D), (out[0], out[1], out[2] > 1, out[3], out[4] > 1), piece


def w4_form(L, dtype, ids, M, N, K, group):
    nt = ctypes.c_int(-1)
    return L.t2sp_gemv_w4_plan(CODES[dtype], ids, M, N, K, group, ctypes.byref(nt)), nt.value


def test_every_form_of_the_grouped_products_has_its_case(lib):
    seen = set()
    for form, types, opb, sizes, K, N in FORWARD:
        for t in types:
            assert forward_form(lib, t, opb, sum(sizes), len(sizes), K, N) == form, (form, t, opb, sum(sizes), len(sizes), K, N)
            seen.add((form, t, opb))
        assert not form[0] or max(sizes) > {16: 2, 32: 16, 64: 32}[form[1]]
    forms = [(True, 16), (True, 32), (True, 64), (False, 64), (False, 128)]
    assert seen == {(f, t, o) for f in forms for t in ALL for o in (0, 1)} | {((False, 256), t, o) for t in BOTH for o in (0, 1)}
    seen = set()
    for tile, parts, types, sizes, K, N in WGRAD:
        for t in types:
            assert wgrad_form(lib, t, sum(sizes), len(sizes), K, N) == (tile, parts), (tile, parts, t)
            seen.add((tile, parts, t))
    assert seen == {(128, p, t) for p in (False, True) for t in ALL} | {(256, False, t) for t in BOTH}


def test_every_form_of_the_cross_entropy_has_its_case(lib):
    seen = set()
    for tile, grad, types, T, V, D in XENT:
        for t in types:
            got = xent_form(lib, t, T, V, D)
            assert got[:2] == (tile, grad), (t, T, V, D, got)
            seen |= {("z", tile, t), ("dH", grad[1], grad[2], t), ("dW", grad[3], grad[4], t)}
    for t in ALL:
        tiles = (64, 128) if t == "float32" else (64, 128, 256)
        assert {("z", tile, t) for tile in tiles} <= seen
        assert {("dH", 128, True, t), ("dW", 128, False, t), ("dW", 128, True, t)} <= seen
    for t in BOTH:
        assert {("dH", 256, True, t), ("dH", 256, False, t), ("dW", 256, False, t)} <= seen


def test_every_form_of_the_4_bit_products_has_its_case(lib):
    seen = set()
    for mt, nt, types, M, N, K, group in W4:
        for t in types:
            assert w4_form(lib, t, 0, M, N, K, group) == (mt, nt), (t, M, N, K, group)
            seen.add((mt, nt, t))
        assert nt == 1 or -(-N // 16) % nt                   # (the last workgroup has tiles behind the last one)
    assert seen == {(m, n, t) for t in BOTH for m, n in ((1, 4), (2, 2), (4, 2), (2, 1), (4, 1))} | \
        {(m, n, "float32") for m, n in ((1, 4), (2, 1), (4, 1), (1, 1))}
    for t in ALL:
        assert w4_form(lib, t, 1, 300, 16397, 296, 32) == (1, 1)


def test_plans_refuse_what_the_calls_refuse(lib):
    i = ctypes.c_int()
    p, five = ctypes.byref(i), (ctypes.c_int * 5)()
    for bad in ((3, 0, 8, 2, 64, 64), (0, 0, 0, 2, 64, 64), (0, 0, 8, 0, 64, 64), (0, 0, 8, 2, 0, 64), (0, 0, 8, 2, 64, 0)):
        assert lib.t2sp_gemm_grouped_plan(*bad, p) == -8
    assert lib.t2sp_gemm_grouped_plan(0, 0, 8, 2, 64, 64, None) == -8 and lib.t2sp_gemm_grouped_wgrad_plan(0, -1, 2, 64, 64, p) == -8
    assert lib.t2sp_gemm_grouped_wgrad_plan(1, 0, 2, 64, 64, p) == 128 and i.value == 1
    assert lib.t2sp_xent_plan(0, 0, 10, 8) == -8 and lib.t2sp_xent_plan(-1, 5, 10, 8) == -8 and lib.t2sp_xent_plan(0, 5, 10, 0) == -8
    assert lib.t2sp_xent_grad_plan(0, 0, 0, 10, 8, five) == -8 and lib.t2sp_xent_grad_plan(0, 0, 5, 10, 8, None) == -8
    assert lib.t2sp_gemv_w4_plan(0, 0, 0, 16, 64, 64, p) == -8 and lib.t2sp_gemv_w4_plan(0, 0, 1, 16, 64, 33, p) == -8


@pytest.mark.parametrize("T,words", [(100, 128001), (8192, 4096), (131072, 4096)])
def test_a_piece_of_the_vocabulary(lib, T, words):
    """128 MB of p - [label], but not fewer than 4096 words."""
    piece = xent_form(lib, "bfloat16", T, 128001, 64)[2]
    assert piece == words and (T * piece * 4 <= 128 << 20 or piece == 4096)
