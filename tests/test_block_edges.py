"""The ends of the norm, routing and tree-norm operators' ranges that need no GPU."""

from __future__ import annotations

import copy

import pytest
import torch

from opaque_amd import _native as N
from opaque_amd import normalization
from opaque_amd.experts import Router
from opaque_amd.normalization import RMSNorm, route_norms

F32, BF16 = N.DTYPE_F32, N.DTYPE_BF16
BAD = 64  # a non-null, aligned address; never read


@pytest.fixture(scope="module")
def lib():
    if not N.LIB_PATH.exists():
        from opaque_amd import build

        build.build()
    return N.load()


def test_an_empty_batch_has_no_gains_and_no_biases(lib):
    norm = lambda n, gains: lib.odp_rms_norm(None, BF16, BF16, BF16, BAD, 8, None, 0, n, 8, BAD, 8, gains, 1e-6, 0.0, 0,
                                             BAD, None, None, None)
    grad = lambda n, gains: lib.odp_rms_norm_grad(None, BF16, BF16, BF16, BAD, 8, BAD, BAD, 8, None, 0, n, 8, BAD, 8, gains,
                                                  0.0, BAD, BAD, None, BAD)
    route = lambda n, biases: lib.odp_route(None, F32, BAD, 8, n, 8, 0, BAD, biases, 1, 1, 0, 2, 1, 1.0, BAD, BAD)
    for call, text in ((norm, "do not divide into"), (grad, "do not divide into"), (route, "do not divide into")):
        assert call(0, 0) == call(0, 3) == N.ODP_OK, N.last_error()
        for n, count in ((4, 0), (4, 3), (0, -1), (4, -2)):
            assert call(n, count) == N.ERR_INVALID_ARGUMENT and text in N.last_error()


def test_gains_of_a_gradient_call_match_the_header():
    text = (N.LIB_PATH.parents[1] / "include" / "opaque_dp.h").read_text()
    assert "ODP_NORM_GRAD_GAINS ((int64_t)1 << 21)" in text and normalization._GRAD_GAINS == 1 << 21


def test_shared_norms_hooks_and_modes_stay():
    """A norm under two names, of one parent and of two, is one norm afterwards too; its hooks run and its mode is kept."""
    net = torch.nn.ModuleDict({"a": torch.nn.RMSNorm(6, eps=1e-3), "c": torch.nn.Sequential(torch.nn.RMSNorm(6))})
    net["b"] = net["a"]
    net["d"] = torch.nn.Sequential(net["a"], net["c"][0])
    net["c"].eval()
    calls, loads = [], []
    handle = net["a"].register_forward_pre_hook(lambda mod, args: calls.append(type(mod)))
    net["a"].register_load_state_dict_pre_hook(lambda mod, *rest: loads.append(type(mod)))
    first, second = net["a"], net["c"][0]
    assert sorted(route_norms(net)) == ["a", "b", "c.0", "d.0", "d.1"]
    assert net["a"] is net["b"] is net["d"][0] is first and net["c"][0] is net["d"][1] is second
    assert all(type(m) is RMSNorm for m in (first, second)) and first.eps == 1e-3 and "eps=0.001" in repr(first)
    assert first.training and not second.training and sum(1 for _ in net.parameters()) == 2
    with pytest.raises(RuntimeError, match="runs on the GPU"):
        net["b"](torch.ones(2, 6))
    net.load_state_dict(net.state_dict())
    assert calls == [RMSNorm] and set(loads) == {RMSNorm}
    handle.remove()
    with pytest.raises(RuntimeError, match="runs on the GPU"):
        net["b"](torch.ones(2, 6))
    assert calls == [RMSNorm] and route_norms(net) == []


def test_norms_that_stay_and_the_model_itself():
    """A module with a forward of its own is not the class's norm; the package's own norms keep their unit offset."""
    net = torch.nn.ModuleDict({"p": torch.nn.RMSNorm(6), "own": RMSNorm(6, unit_offset=True)})
    net["p"].forward = lambda x: x
    assert route_norms(net, (torch.nn.RMSNorm, RMSNorm)) == [] and net["own"].unit_offset
    assert type(net["p"]) is torch.nn.RMSNorm
    alone = torch.nn.RMSNorm(6)
    assert route_norms(alone) == [""] and type(alone) is RMSNorm
    without = torch.nn.Linear(6, 1)  # no eps: an error before anything changes
    without.weight = torch.nn.Parameter(torch.ones(6))
    both = torch.nn.Sequential(torch.nn.RMSNorm(6), without)
    with pytest.raises(AttributeError):
        route_norms(both, (torch.nn.RMSNorm, torch.nn.Linear))
    assert type(both[0]) is torch.nn.RMSNorm


@pytest.mark.parametrize("cast", [lambda m: m.to(torch.bfloat16), lambda m: m.half(), lambda m: m.double(),
                                  lambda m: m.to(torch.bfloat16).float(), lambda m: m.to("cpu", torch.bfloat16),
                                  lambda m: copy.deepcopy(m).bfloat16()],
                         ids=["bfloat16", "half", "double", "back", "device", "copy"])
def test_a_routers_bias_stays_float32(cast):
    """Steps below a narrow type's resolution survive a cast of the model, and of the router itself."""
    net = torch.nn.Sequential(torch.nn.Linear(8, 8), Router(8, 4, 2, balance=True))
    step = torch.tensor([1.0, -1.0, 0.5, 0.0]) + 1e-5
    net[1].balance += step
    got = cast(net)
    assert got[1].balance.dtype == torch.float32 and torch.equal(got[1].balance, step)
    assert got[1].weight.dtype == got[0].weight.dtype and set(dict(got.named_buffers())) == {"1.balance"}
    assert torch.equal(cast(Router(8, 4, 2, balance=True)).balance, torch.zeros(4))
    assert cast(Router(8, 4, 2)).balance is None


def test_a_routers_bias_is_float32_from_the_start():
    before = torch.get_default_dtype()
    try:
        torch.set_default_dtype(torch.bfloat16)
        assert Router(8, 4, 2, balance=True).balance.dtype == torch.float32
    finally:
        torch.set_default_dtype(before)
    meta = Router(8, 4, 2, balance=True, device="meta", dtype=torch.bfloat16).to_empty(device="cpu")
    assert meta.balance.dtype == torch.float32 and meta.weight.dtype == torch.bfloat16
