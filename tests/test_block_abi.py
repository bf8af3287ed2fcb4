"""Refusals of the norm, routing and tree-norm operators: C entry points and Python calls (no GPU: every call returns
before device work)."""

from __future__ import annotations

import ctypes

import pytest
import torch

from opaque_amd import _native as N
from opaque_amd.experts import Router, route
from opaque_amd.global_norm import clip_by_global_norm, global_norm
from opaque_amd.normalization import RMSNorm, rms_norm, rms_norm_quantized, route_norms
from opaque_amd.types import SecondMomentNoiseOutput, clipped, noised

F32, BF16, F16, F64 = N.DTYPE_F32, N.DTYPE_BF16, N.DTYPE_F16, N.DTYPE_F64
BAD = 64  # a non-null, aligned address; never read


@pytest.fixture(scope="module")
def lib():
    if not N.LIB_PATH.exists():
        from opaque_amd import build

        build.build()
    return N.load()


def refused(rc, status, text):
    assert rc == status and text in N.last_error(), (rc, N.last_error())


def test_norm_checks(lib):
    norm = lambda dt=BF16, ht=BF16, gt=BF16, x=BAD, ldx=8, r=None, ldr=8, n=4, d=8, g=BAD, ldg=0, gains=1, q=0, y=BAD, \
        h=None, s=None: lib.odp_rms_norm(None, dt, ht, gt, x, ldx, r, ldr, n, d, g, ldg, gains, 1e-6, 0.0, q, y, h, None, s)
    for kw in ({"dt": F64, "ht": F64, "gt": F64}, {"ht": F16}, {"gt": F16}, {"dt": F32}):
        refused(norm(**kw), N.ERR_UNSUPPORTED, "types")
    for kw in ({"n": -1}, {"n": 1 << 31}, {"d": 0}, {"d": 32769, "ldx": 32769}):
        refused(norm(**kw), N.ERR_INVALID_ARGUMENT, "fewer than 2^31 rows")
    for kw in ({"gains": 0}, {"gains": 3}, {"gains": 8}):
        refused(norm(**kw), N.ERR_INVALID_ARGUMENT, "do not divide")
    for kw in ({"q": 3, "s": BAD}, {"q": -1}):
        refused(norm(**kw), N.ERR_INVALID_ARGUMENT, "quant")
    for kw in ({"x": None}, {"y": None}, {"r": BAD}, {"h": BAD}, {"q": 1}, {"s": BAD}):
        refused(norm(**kw), N.ERR_INVALID_ARGUMENT, "null x or y")
    for kw in ({"ldx": 7}, {"r": BAD, "h": BAD, "ldr": 7}, {"ldg": 4}, {"ldx": -8}):
        refused(norm(**kw), N.ERR_INVALID_ARGUMENT, "pitch")
    assert norm(n=0, x=None, y=None) == N.ODP_OK


def test_norm_gradient_checks(lib):
    grad = lambda dt=BF16, ht=BF16, gt=F32, h=BAD, ldh=8, rs=BAD, gy=BAD, ldy=8, gh=None, ldgh=0, n=4096, d=8, g=BAD, \
        ldg=0, gains=1, scr=BAD, dx=BAD, dr=None, dg=BAD: lib.odp_rms_norm_grad(
            None, dt, ht, gt, h, ldh, rs, gy, ldy, gh, ldgh, n, d, g, ldg, gains, 0.0, scr, dx, dr, dg)
    refused(grad(dt=F64), N.ERR_UNSUPPORTED, "types")
    refused(grad(n=-1), N.ERR_INVALID_ARGUMENT, "rows")
    refused(grad(gains=5), N.ERR_INVALID_ARGUMENT, "do not divide")
    for kw in ({"h": None}, {"rs": None}, {"gy": None}, {"dx": None, "dr": BAD}):
        refused(grad(**kw), N.ERR_INVALID_ARGUMENT, "null h, rstd or gy")
    for kw in ({"ldh": 4}, {"ldy": 4}, {"gh": BAD, "ldgh": 4}, {"ldg": 4}):
        refused(grad(**kw), N.ERR_INVALID_ARGUMENT, "pitch")
    refused(grad(scr=None), N.ERR_INVALID_ARGUMENT, "scratch")
    refused(grad(n=1 << 24, gains=1 << 24), N.ERR_UNSUPPORTED, "more than one launch")
    assert grad(n=0, gains=1, h=None, rs=None, gy=None) == N.ODP_OK
    assert grad(dx=None, dg=None) == N.ODP_OK
    scratch = lib.odp_rms_norm_grad_scratch
    assert scratch(0, 8, 1) == scratch(4, 0, 1) == scratch(4, 8, 0) == scratch(4, 8, 3) == 0
    assert scratch(1, 4096, 1) == scratch(4096, 4096, 4096) == 0
    for n, d, gains in ((4096, 4096, 1), (16384, 4096, 16), (100000, 64, 1), (777, 1001, 1), (1 << 30, 32768, 2)):
        assert scratch(n, d, gains) % (4 * gains * d) == 0 and 0 < scratch(n, d, gains) <= 4 * d * (1024 + gains)


def test_route_checks(lib):
    route_ = lambda dt=F32, z=BAD, ldz=64, n=4, e=64, sig=0, b=None, nb=1, g=1, tg=1, best=0, k=8, sc=1.0, idx=BAD, w=BAD: \
        lib.odp_route(None, dt, z, ldz, n, e, sig, b, nb, g, tg, best, k, 1, sc, idx, w)
    refused(route_(dt=F64), N.ERR_UNSUPPORTED, "dtype")
    for kw in ({"n": -1}, {"n": 1 << 31}, {"e": 0}, {"e": 1025, "ldz": 1025}, {"k": 0}, {"k": 65}, {"e": 4, "k": 5},
               {"ldz": 63}):
        refused(route_(**kw), N.ERR_INVALID_ARGUMENT, "invalid sizes")
    for kw in ({"g": 0}, {"g": 5}, {"g": 65, "e": 65, "ldz": 65, "k": 1}, {"g": 8, "tg": 9}, {"g": 8, "tg": 0}, {"best": 2},
               {"g": 16, "tg": 1, "k": 5}):
        refused(route_(**kw), N.ERR_INVALID_ARGUMENT, "groups")
    for nb in (0, 3):
        refused(route_(b=BAD, nb=nb), N.ERR_INVALID_ARGUMENT, "biases")
    for sc in (float("inf"), float("nan")):
        refused(route_(sc=sc), N.ERR_INVALID_ARGUMENT, "scale")
    for kw in ({"z": None}, {"idx": None}, {"w": None}):
        refused(route_(**kw), N.ERR_INVALID_ARGUMENT, "null pointer")
    assert route_(n=0, z=None, idx=None, w=None) == N.ODP_OK
    grad = lambda dt=F32, z=BAD, ldz=64, n=4, e=64, k=8, idx=BAD, gw=BAD, ldw=8, dz=BAD: lib.odp_route_grad(
        None, dt, z, ldz, n, e, 0, k, 1, 1.0, idx, gw, ldw, dz)
    refused(grad(dt=F64), N.ERR_UNSUPPORTED, "dtype")
    refused(grad(k=65), N.ERR_INVALID_ARGUMENT, "invalid sizes")
    for kw in ({"z": None}, {"idx": None}, {"gw": None}, {"dz": None}, {"ldw": -1}):
        refused(grad(**kw), N.ERR_INVALID_ARGUMENT, "null pointer")
    assert grad(n=0, z=None) == N.ODP_OK


def test_tree_checks(lib):
    def tree(rows, clip=1, most=1.0, scratch=BAD, norm=BAD, n=None):
        table = (ctypes.c_int64 * (4 * len(rows)))(*[v for r in rows for v in r])
        return lib.odp_tree_norm(None, ctypes.addressof(table) if rows else None, len(rows) if n is None else n, clip, most,
                                 0, scratch, norm)

    ok = [BAD, BAD, 4, F32]
    for kw in ({"scratch": None}, {"norm": None}, {"n": -1}):
        refused(tree([ok], **kw), N.ERR_INVALID_ARGUMENT, "null pointer")
    refused(lib.odp_tree_norm(None, None, 2, 1, 1.0, 0, BAD, BAD), N.ERR_INVALID_ARGUMENT, "null pointer")
    for most in (-1.0, float("nan")):
        refused(tree([ok], most=most), N.ERR_INVALID_ARGUMENT, "max_norm")
    for n in (-1, (1 << 44) + 1):
        refused(tree([ok, [BAD, BAD, n, F32]]), N.ERR_INVALID_ARGUMENT, "leaf 1 has")
    for dt in (-1, 4):
        refused(tree([[BAD, BAD, 4, dt]]), N.ERR_UNSUPPORTED, "dtype")
    for row in ([0, BAD, 4, F32], [BAD, 0, 4, F32]):
        refused(tree([ok, row]), N.ERR_INVALID_ARGUMENT, "leaf 1 has a null")
    assert lib.odp_tree_norm_scratch(0) == 8 and lib.odp_tree_norm_scratch(128) * 2 == lib.odp_tree_norm_scratch(129)


def test_the_table_matches_the_header():
    text = (N.LIB_PATH.parents[1] / "include" / "opaque_dp.h").read_text()
    assert "ODP_TN_SRC = 0, ODP_TN_DST, ODP_TN_N, ODP_TN_DTYPE, ODP_TN_FIELDS = 4" in text and N.TN_FIELDS == 4
    assert (N.TN_SRC, N.TN_DST, N.TN_N, N.TN_DTYPE) == (0, 1, 2, 3)
    from opaque_amd import experts, normalization

    assert f"ODP_NORM_WIDE ((int64_t){normalization._WIDE})" in text
    assert f"ODP_ROUTE_EXPERTS {experts._EXPERTS}" in text and f"ODP_ROUTE_CHOICES {experts._CHOICES}" in text


@pytest.mark.parametrize("call", [rms_norm, rms_norm_quantized])
def test_norm_refusals(call):
    x = torch.ones(3, 8)
    w = torch.ones(8)
    for bad in ([1.0], x.double(), x.int()):
        with pytest.raises(TypeError, match="supports"):
            call(bad)
    for bad in (torch.tensor(1.0), torch.ones(3, 0), torch.ones(1, 32769)):
        with pytest.raises(ValueError, match="rows of 1 to"):
            call(bad)
    for bad in (torch.ones(7), torch.ones(1, 8), torch.ones(3, 8)):
        with pytest.raises(ValueError, match="weight must be"):
            call(x, bad)
    for t in (torch.float64, torch.bfloat16):
        with pytest.raises(TypeError, match="weight must be"):
            call(x, w.to(t))
        with pytest.raises(TypeError, match="residual must be"):
            call(x, w, residual=x.to(t))
    with pytest.raises(TypeError, match="residual must be"):
        call(x.half(), w, residual=x.bfloat16())
    with pytest.raises(ValueError, match="residual must be"):
        call(x, w, residual=x[:2])
    with pytest.raises(RuntimeError, match="runs on the GPU"):
        call(x, w, residual=x)


def test_route_refusals():
    z = torch.ones(3, 8)
    for bad in ([1.0], z.double(), z.int()):
        with pytest.raises(TypeError, match="supports"):
            route(bad, 2)
    for bad in (torch.tensor(1.0), torch.ones(3, 0), torch.ones(1, 1025)):
        with pytest.raises(ValueError, match="logits of 1 to"):
            route(bad, 1)
    for kw, text in (({"scores": "tanh"}, "scores"), ({"group_best": "sum"}, "group_best"), ({"groups": 3}, "groups"),
                     ({"groups": 0}, "groups"), ({"groups": 4, "top_groups": 5}, "groups"), ({"top_groups": 0}, "groups")):
        with pytest.raises(ValueError, match=text):
            route(z, 2, **kw)
    for k in (0, 9, -1):
        with pytest.raises(ValueError, match="top_k"):
            route(z, k)
    with pytest.raises(ValueError, match="top_k"):
        route(z, 3, groups=4, top_groups=1)
    with pytest.raises(ValueError, match="top_k"):
        route(torch.ones(3, 100), 65)
    for bad in (torch.ones(7), torch.ones(3, 8)):
        with pytest.raises(ValueError, match="bias must be"):
            route(z, 2, bias=bad)
    with pytest.raises(TypeError, match="bias must be"):
        route(z, 2, bias=torch.ones(8, dtype=torch.bfloat16))
    with pytest.raises(RuntimeError, match="runs on the GPU"):
        route(z, 2)


def test_tree_refusals():
    for call in (global_norm, lambda t: clip_by_global_norm(t, 1.0)):
        with pytest.raises(RuntimeError, match="run on the GPU|runs on the GPU"):
            call({"a": torch.ones(3)})
        for t in (torch.ones(3, dtype=torch.int32), torch.ones(3, dtype=torch.complex64)):
            with pytest.raises(TypeError, match="supports"):
                call([t])
    for bad in (-1.0, float("nan")):
        with pytest.raises(ValueError, match="max_norm"):
            clip_by_global_norm({}, bad)
    with pytest.raises(TypeError, match="add the noise"):
        clip_by_global_norm(clipped({}, max_norm=1.0), 1.0)
    pair = SecondMomentNoiseOutput(*(noised({}, max_norm=1.0, noise_stddev=1.0) for _ in range(2)))
    for call in (global_norm, lambda t: clip_by_global_norm(t, 1.0)):
        with pytest.raises(TypeError, match="by itself"):
            call(pair)
    got, norm = clip_by_global_norm({"a": None, "b": [3]}, 1.0)
    assert got == {"a": None, "b": [3]} and float(norm) == 0


def test_modules_on_the_host():
    """Modules are made, saved and loaded anywhere; only their calls need the GPU."""
    m = RMSNorm(12, eps=1e-5)
    assert m.weight.shape == (12,) and bool((m.weight == 1).all()) and "eps=1e-05" in repr(m)
    r = Router(12, 8, 2, balance=True, dtype=torch.bfloat16)
    assert r.weight.shape == (8, 12) and r.balance.dtype == torch.float32
    assert set(r.state_dict()) == {"weight", "balance"} and Router(12, 8, 2).balance is None
    Router(12, 8, 2, balance=True).load_state_dict({k: v.float() for k, v in r.state_dict().items()})


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_the_default_eps_is_torchs(dtype):
    """By what torch gives for rows whose mean square lies between the types' eps."""
    net = torch.nn.Sequential(torch.nn.RMSNorm(64, dtype=dtype))
    x = (1e-3 * torch.randn(8, 64, generator=torch.Generator().manual_seed(0))).to(dtype)
    y = net(x).detach().double()
    route_norms(net)
    want = x.double() / torch.sqrt(x.double().square().mean(1, keepdim=True) + net[0].eps)
    # Half a step of the type for each of x's norm and the gain's product, and float32's sum.
    assert ((y - want).abs() <= (torch.finfo(dtype).eps + 80 * 2.0**-24) * want.abs()).all()


def test_norms_are_replaced_on_their_own_gains():
    class Other(torch.nn.Module):  # the layout of Hugging Face's
        def __init__(self):
            super().__init__()
            self.weight, self.variance_epsilon = torch.nn.Parameter(torch.ones(6)), 1e-5

    inner = torch.nn.Sequential(torch.nn.RMSNorm(6, eps=1e-4), torch.nn.Linear(6, 6), Other())
    net = torch.nn.ModuleDict({"a": torch.nn.RMSNorm(6), "b": inner, "c": torch.nn.RMSNorm((2, 6)),
                               "d": torch.nn.RMSNorm(6, elementwise_affine=False)})
    kept = {k: v for k, v in net.named_parameters()}
    assert route_norms(net, (torch.nn.RMSNorm, Other)) == ["a", "b.0", "b.2"]
    assert {k: id(v) for k, v in net.named_parameters()} == {k: id(v) for k, v in kept.items()}
    assert [net["a"].eps, net["b"][0].eps, net["b"][2].eps] == [torch.finfo(torch.float32).eps, 1e-4, 1e-5]
    assert type(net["c"]) is type(net["d"]) is torch.nn.RMSNorm and type(net["b"][2]) is RMSNorm
