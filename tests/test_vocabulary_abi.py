"""Argument checks and size helpers of the vocabulary operators' C entry points (no GPU: every call returns before device work)."""

from __future__ import annotations

import pytest

from opaque_amd import _native as N

F32, BF16, F16, F64 = N.DTYPE_F32, N.DTYPE_BF16, N.DTYPE_F16, N.DTYPE_F64
BAD = 64  # a non-null, aligned address; never read
BIG = 1 << 31


@pytest.fixture(scope="module")
def lib():
    if not N.LIB_PATH.exists():
        from opaque_amd import build

        build.build()
    return N.load()


def refused(rc, status, text):
    assert rc == status and text in N.last_error(), (rc, N.last_error())


def test_embedding_checks(lib):
    rows = lambda dt=F32, y=BAD, tb=8, n=4, w=BAD, ldw=8, v=10, d=8, out=BAD: lib.odp_embed_rows(
        None, dt, y, tb, n, w, ldw, v, d, 1.0, out)
    refused(rows(dt=F64), N.ERR_UNSUPPORTED, "dtype 3")
    refused(rows(tb=2), N.ERR_UNSUPPORTED, "tokens of 2 bytes")
    for kw in ({"n": -1}, {"n": BIG}, {"d": 0}, {"d": 1 << 24, "ldw": 1 << 24}, {"v": 0}, {"v": BIG}, {"ldw": 7}):
        refused(rows(**kw), N.ERR_INVALID_ARGUMENT, "invalid sizes")
    for kw in ({"y": None}, {"w": None}, {"out": None}):
        refused(rows(**kw), N.ERR_INVALID_ARGUMENT, "null pointer")
    refused(rows(n=1 << 30, d=1 << 20, ldw=1 << 20), N.ERR_UNSUPPORTED, "workgroups")
    assert rows(n=0, y=None, w=None, out=None) == N.ODP_OK


def test_sort_checks(lib):
    sort = lambda y=BAD, tb=8, n=4, v=10, ss=None, sl=None, ns=0, scr=BAD, k=BAD, r=BAD, so=None, z=None, zb=0: \
        lib.odp_token_sort(None, y, tb, n, v, -1, ss, sl, ns, scr, k, r, so, z, zb)
    refused(sort(tb=1), N.ERR_UNSUPPORTED, "tokens of 1 bytes")
    refused(sort(v=0), N.ERR_INVALID_ARGUMENT, "invalid sizes")
    refused(sort(zb=-1), N.ERR_INVALID_ARGUMENT, "-1 bytes")
    for kw in ({"y": None}, {"scr": None}, {"scr": 8}, {"k": None}, {"r": None}, {"ns": -1}, {"ss": BAD, "so": BAD},
               {"ss": BAD, "sl": BAD}):
        refused(sort(**kw), N.ERR_INVALID_ARGUMENT, "odp_token_sort: null pointer")
    assert sort(n=0, y=None, scr=None, k=None, r=None) == N.ODP_OK
    assert lib.odp_token_sort_scratch(0, 10) == 0 and lib.odp_token_sort_scratch(5, 0) == 0
    assert lib.odp_token_sort_scratch(100, 10) >= 4 * 300
    assert lib.odp_token_sort_scratch(1 << 20, 10) > 4 * 3 * (1 << 20)


def test_embedding_sum_checks(lib):
    grad = lambda dt=BF16, g=BAD, ldg=8, n=4, k=BAD, r=BAD, scr=BAD, out=BAD: lib.odp_embed_grad(
        None, dt, g, ldg, n, 8, k, r, 10, 1.0, scr, out)
    norm = lambda g=BAD, n=4, ss=BAD, w=BAD, part=BAD, stride=4, slot=0, nf=BAD: lib.odp_embed_sqnorm(
        None, BF16, g, 8, n, 8, BAD, BAD, BAD, 10, 1.0, ss, BAD, BAD, w, part, stride, slot, nf)
    clip = lambda g=BAD, n=4, od=F32, out=BAD, sc=BAD: lib.odp_embed_clipped_sum(
        None, BF16, g, 8, n, 8, BAD, BAD, BAD, 10, 1.0, BAD, BAD, BAD, sc, 1.0, od, out, None)
    refused(grad(dt=F64), N.ERR_UNSUPPORTED, "dtype 3")
    refused(grad(ldg=7), N.ERR_INVALID_ARGUMENT, "invalid sizes")
    for kw in ({"g": None}, {"k": None}, {"r": None}, {"scr": None}, {"out": None}, {"out": None, "n": 0}):
        refused(grad(**kw), N.ERR_INVALID_ARGUMENT, "odp_embed_grad: null pointer")
    for kw in ({"g": None}, {"ss": None}, {"w": None}, {"part": None}, {"nf": None}, {"slot": 4}, {"slot": -1}):
        refused(norm(**kw), N.ERR_INVALID_ARGUMENT, "odp_embed_sqnorm")
    refused(clip(od=4), N.ERR_UNSUPPORTED, "out_dtype 4")
    for kw in ({"g": None}, {"out": None}, {"sc": None}):
        refused(clip(**kw), N.ERR_INVALID_ARGUMENT, "odp_embed_clipped_sum: null pointer")
    assert grad(n=0, g=None) == norm(n=0, g=None) == clip(n=0, g=None) == N.ODP_OK
    assert [lib.odp_embed_pieces(F32, d) for d in (0, 1, 256, 257)] == [0, 1, 1, 2]
    assert [lib.odp_embed_pieces(BF16, d) for d in (1, 512, 513)] == [1, 1, 2]
    one, two = (lib.odp_embed_sum_scratch(BF16, 1000, 600, k) for k in (0, 1))
    assert two == 2 * one > 0 and lib.odp_embed_sum_scratch(BF16, 0, 600, 0) == 0


def test_loss_checks(lib):
    rows = lambda dt=BF16, x=BAD, ldx=8, n=4, cols=8, width=8, y=BAD, tb=8, v=10, xc=BAD, cnt=BAD: lib.odp_xent_rows(
        None, dt, x, ldx, n, cols, width, y, tb, v, -100, 0, xc, BAD, BAD, BAD, cnt, BAD, BAD)
    refused(rows(dt=F16), N.ERR_UNSUPPORTED, "dtype 2")
    for kw in ({"n": -1}, {"n": BIG - 512}, {"width": 12, "cols": 12, "ldx": 12}, {"width": 0}, {"v": 0},
               {"v": BIG - 512}, {"width": 1 << 20}):
        refused(rows(**kw), N.ERR_INVALID_ARGUMENT, "invalid sizes")
    for kw in ({"cols": 9}, {"cols": 0}, {"ldx": 7}, {"tb": 2}):
        refused(rows(**kw), N.ERR_INVALID_ARGUMENT, "columns of pitch")
    for kw in ({"x": None}, {"y": None}, {"xc": None}, {"cnt": None}, {"xc": 8}):
        refused(rows(**kw), N.ERR_INVALID_ARGUMENT, "null")

    losses = lambda dt=BF16, xc=BAD, n=4, ldw=8, w=BAD, v=10, scr=BAD, z=None, ldl=0: lib.odp_xent_losses(
        None, dt, xc, n, 8, BAD, BAD, BAD, w, ldw, v, 0.0, scr, BAD, BAD, z, ldl)
    refused(losses(dt=F16), N.ERR_UNSUPPORTED, "dtype 2")
    for ldw in (4, 12, 1 << 20):
        refused(losses(ldw=ldw), N.ERR_INVALID_ARGUMENT, "invalid sizes")
    for kw in ({"xc": None}, {"w": None}, {"scr": None}, {"w": 8}, {"xc": 8}):
        refused(losses(**kw), N.ERR_INVALID_ARGUMENT, "null pointer, or rows off")
    for kw in ({"z": BAD, "ldl": 10}, {"z": 8, "ldl": 256}):
        refused(losses(**kw), N.ERR_INVALID_ARGUMENT, "logits of pitch")
    refused(losses(n=1 << 30, v=1 << 30), N.ERR_UNSUPPORTED, "tiles")
    assert losses(n=0, xc=None) == N.ODP_OK
    refused(lib.odp_xent_reduce(None, BAD, 4, None, None), N.ERR_INVALID_ARGUMENT, "null pointer")
    refused(lib.odp_xent_reduce(None, None, 4, None, BAD), N.ERR_INVALID_ARGUMENT, "null pointer")


def test_loss_gradient_checks(lib):
    dlogits = lambda n=4, v0=0, vc=10, z=None, ldl=0, dl=BAD, ldd=256, rest=BAD, v=600: lib.odp_xent_dlogits(
        None, BF16, BAD, n, 8, BAD, BAD, BAD, BAD, 8, v, 0.0, v0, vc, BAD, BAD, 1, None, z, ldl, dl, ldd, rest)
    for kw in ({"v0": -1}, {"vc": 0}, {"v0": 591}, {"ldd": 10}):
        refused(dlogits(**kw), N.ERR_INVALID_ARGUMENT, "columns [")
    for kw in ({"dl": None}, {"dl": 8}, {"rest": None}):
        refused(dlogits(**kw), N.ERR_INVALID_ARGUMENT, "null pointer, or rows off")
    for kw in ({"z": BAD, "ldl": 600}, {"z": 8, "ldl": 768}, {"z": BAD, "ldl": 768, "v0": 8}):
        refused(dlogits(**kw), N.ERR_INVALID_ARGUMENT, "logits of pitch")
    assert dlogits(n=0, dl=None) == N.ODP_OK

    dx = lambda n=4, v0=0, vc=10, piece=10, w=BAD, dl=BAD, ldd=256, scr=BAD: lib.odp_xent_dx(
        None, BF16, n, 8, BAD, w, 8, 600, v0, vc, piece, dl, ldd, scr)
    for kw in ({"vc": 11}, {"v0": 595}, {"ldd": 10}):
        refused(dx(**kw), N.ERR_INVALID_ARGUMENT, "in pieces of")
    for kw in ({"w": None}, {"dl": None}, {"scr": None}, {"scr": 8}):
        refused(dx(**kw), N.ERR_INVALID_ARGUMENT, "null pointer, or rows off")
    rows = lambda n=4, cols=8, piece=10, scr=BAD, out=BAD: lib.odp_xent_dx_rows(
        None, BF16, n, cols, 8, BAD, BAD, BAD, BAD, 8, piece, scr, BAD, out)
    for kw in ({"cols": 9}, {"cols": 0}, {"piece": 0}):
        refused(rows(**kw), N.ERR_INVALID_ARGUMENT, "pieces of")
    for kw in ({"scr": None}, {"out": None}, {"out": 8}):
        refused(rows(**kw), N.ERR_INVALID_ARGUMENT, "null pointer, or rows off")

    dw = lambda n=4, xc=BAD, vc=10, dl=BAD, ldd=256, scr=None, out=BAD, lddw=8: lib.odp_xent_dw(
        None, BF16, xc, n, 8, BAD, vc, dl, ldd, scr, out, lddw)
    for kw in ({"ldd": 10}, {"xc": None}, {"dl": None}, {"out": None}, {"out": 8}):
        refused(dw(**kw), N.ERR_INVALID_ARGUMENT, "odp_xent_dw: pitch")
    refused(dw(lddw=4), N.ERR_INVALID_ARGUMENT, "invalid sizes")
    assert lib.odp_xent_dw_scratch(BF16, 65536, 10, 8) > 0
    refused(dw(n=65536), N.ERR_INVALID_ARGUMENT, "scratch is null")


def test_loss_sizes(lib):
    assert [lib.odp_xent_pitch(BF16, c) for c in (0, 1, 256, 257)] == [0, 256, 256, 512]
    assert [lib.odp_xent_pitch(F32, c) for c in (1, 128, 129)] == [128, 128, 256]
    assert lib.odp_xent_kept(BF16, 4096, 1024, 1000) == 4 * 4096 * 1024
    assert lib.odp_xent_kept(BF16, 4096, 64, 1000) == 0  # forming them again is faster
    assert lib.odp_xent_kept(F32, 4096, 128, 1000) == 4 * 4096 * 1024
    assert lib.odp_xent_kept(BF16, 16, 64, 1000) == 4 * 16 * 1024
    assert lib.odp_xent_stats_scratch(BF16, 1000, 512) == 4 * 1000 * (2 * 2 + 1)
    for n, width in ((1, 64), (64, 4096), (65, 8), (5000, 1000)):
        assert lib.odp_xent_dx_scratch(BF16, n, width) >= 4 * n * width
    # Slices of the tokens where the tiles of dW are few, none where they fill the CUs.
    assert lib.odp_xent_dw_scratch(BF16, 8192, 256, 512) == 4 * 8 * 256 * 512
    assert lib.odp_xent_dw_scratch(BF16, 8192, 64256, 4096) == lib.odp_xent_dw_scratch(BF16, 1000, 256, 512) == 0
    assert lib.odp_xent_dw_scratch(F32, 65536, 100, 64) == 4 * 128 * 100 * 64
