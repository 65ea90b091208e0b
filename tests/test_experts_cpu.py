"""Routing and the experts' products, what needs no GPU: refusals at the C boundary, before any launch, and of the Python entry points."""
import ctypes as C

import pytest
import torch

from ixrun_amd import _lib, route_experts


def _routing(**change):
    r = _lib.IxhRouting(16, 4, 4, 2, 0, 1, 1.0)
    for k, v in change.items():
        setattr(r, k, v)
    return r


@pytest.mark.parametrize("change,needle", [
    ({"experts": 0}, "not in 1..1024"),
    ({"experts": 1025}, "not in 1..1024"),
    ({"top_k": 0}, "top_k"),
    ({"top_k": 17}, "top_k"),
    ({"experts": 128, "top_k": 65, "n_groups": 1, "top_groups": 1}, "top_k"),
    ({"n_groups": 3}, "equal length"),
    ({"n_groups": 0}, "equal length"),
    ({"experts": 130, "n_groups": 65}, "groups"),
    ({"top_groups": 0}, "top_groups"),
    ({"top_groups": 5}, "top_groups"),
    ({"top_groups": 1, "top_k": 5}, "best groups have"),
    ({"scoring": 2}, "scoring"),
])
def test_malformed_routings_are_refused(change, needle):
    lib = _lib.lib()
    r = _routing(**change)
    assert lib.ixh_route(C.byref(r), 0x1000, 0, 2048, 3, None, 0x1000, 0x1000, None) == -1
    assert needle in lib.ixh_last_error().decode()


@pytest.mark.parametrize("arguments,needle", [
    (dict(dtype=3), "dtype"), (dict(logits=None), "NULL"), (dict(ids=None), "NULL"), (dict(weights=None), "NULL"), (dict(ld=15), "ld"),
    (dict(tokens=-1), "tokens"), (dict(tokens=1 << 30), "tokens"),
])
def test_malformed_routing_calls_are_refused(arguments, needle):
    lib = _lib.lib()
    a = dict(dict(logits=0x1000, dtype=0, ld=16, tokens=2, ids=0x1000, weights=0x1000), **arguments)
    assert lib.ixh_route(C.byref(_routing()), a["logits"], a["dtype"], a["ld"], a["tokens"], None, a["ids"], a["weights"], None) == -1
    assert needle in lib.ixh_last_error().decode()


def test_no_tokens_launch_nothing():
    assert _lib.lib().ixh_route(C.byref(_routing()), None, 0, 16, 0, None, None, None, None) == 0
    assert _lib.lib().ixh_experts(C.byref(_experts()), None, 0, 0, None, None, 2, None, 0, None, 0, None, 0, None) == 0


def _matrix(out_f, in_f, experts=4, bits=4):
    words = _lib.lib().ixh_lanes_plane_words(out_f, in_f, bits)
    return _lib.IxhExpertMatrix(bits, out_f, in_f, 0x1000, words * experts, 0x1000, 0x1000, 0x1000, 64 * experts, 0x1000, None)


def _experts(hidden=96, inner=40, gated=1):
    rows = (inner + 15) // 16 * 32 if gated else inner
    return _lib.IxhExperts(4, gated, 1, hidden, inner, _matrix(rows, hidden), _matrix(hidden, inner))


@pytest.mark.parametrize("change,needle", [
    (lambda e: setattr(e, "n_experts", 0), "not in 1..1024"),
    (lambda e: setattr(e, "n_experts", 1025), "not in 1..1024"),
    (lambda e: setattr(e, "n_experts", 5), "planes of"),
    (lambda e: setattr(e, "hidden", 0), "experts: 40 x 0"),
    (lambda e: setattr(e, "activation", 6), "activation"),
    (lambda e: setattr(e, "inner", 48 + 16), "the first matrix"),
    (lambda e: setattr(e, "gated", 0), "the first matrix"),
    (lambda e: setattr(e.second, "in_f", 41), "the second matrix"),
    (lambda e: setattr(e.first, "bits", 6), "no lane layout"),
    (lambda e: setattr(e.first, "plane", 0x1004), "16-byte"),
    (lambda e: setattr(e.second, "scale", None), "scale"),
    (lambda e: setattr(e.second, "exc_off", None), "scale"),
    (lambda e: setattr(e.second, "n_quads", 65), "groups of 64"),
    (lambda e: setattr(e.second, "n_quads", 1 << 30), "groups of 64"),
    (lambda e: setattr(e, "hidden", 1 << 24), "experts: 40 x 16777216"),
    (lambda e: setattr(e.second, "exc_pos", 0x1004), "8-byte"),
    (lambda e: setattr(e.first, "exc_val", 0x1002), "aligned"),
    (lambda e: setattr(e.first, "exc_off", 0x1002), "aligned"),
])
def test_malformed_experts_are_refused(change, needle):
    lib = _lib.lib()
    e = _experts()
    assert lib.ixh_experts_workspace_bytes(C.byref(e), 3, 2) > 0
    change(e)
    assert lib.ixh_experts_workspace_bytes(C.byref(e), 3, 2) == 0
    assert lib.ixh_experts(C.byref(e), 0x1000, 96, 3, 0x1000, 0x1000, 2, None, 0, 0x1000, 96, 0x1000, 1 << 40, None) == -1
    assert needle in lib.ixh_last_error().decode()


@pytest.mark.parametrize("arguments,code,needle", [
    (dict(x=None), -1, "NULL"), (dict(ids=None), -1, "NULL"), (dict(weights=None), -1, "NULL"), (dict(y=None), -1, "NULL"),
    (dict(ldx=95), -1, "shorter"), (dict(ldy=95), -1, "shorter"), (dict(residual=0x1000, ld_residual=95), -1, "shorter"),
    (dict(tokens=-1), -1, "2^20"), (dict(tokens=(1 << 19) + 1), -1, "2^20"), (dict(top_k=0), -1, "2^20"),
    (dict(ws=None), -4, "workspace"), (dict(ws_bytes=16), -4, "workspace"),
])
def test_malformed_experts_calls_are_refused(arguments, code, needle):
    lib = _lib.lib()
    a = dict(dict(x=0x1000, ldx=96, tokens=3, ids=0x1000, weights=0x1000, top_k=2, residual=None, ld_residual=0, y=0x1000, ldy=96, ws=0x1000,
                  ws_bytes=1 << 40), **arguments)
    e = _experts()
    assert lib.ixh_experts(C.byref(e), a["x"], a["ldx"], a["tokens"], a["ids"], a["weights"], a["top_k"], a["residual"], a["ld_residual"], a["y"],
                           a["ldy"], a["ws"], a["ws_bytes"], None) == code
    assert needle in lib.ixh_last_error().decode()


def test_python_refuses_what_is_not_on_the_gpu_or_has_a_gradient():
    with pytest.raises(RuntimeError, match="GPU"):
        route_experts(torch.zeros(2, 8), 2)
    with pytest.raises(RuntimeError, match="no gradient"):
        route_experts(torch.zeros(2, 8, requires_grad=True), 2)


def test_dual_tensors_are_refused_wherever_they_live():
    from torch.autograd import forward_ad

    x = torch.zeros(2, 4)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, x + 1)
        for grad in (torch.enable_grad, torch.no_grad):
            with grad():
                _lib.inference_only("this", x, None, torch.zeros(3, dtype=torch.int32))
                with pytest.raises(RuntimeError, match="this has no gradient"):
                    _lib.inference_only("this", x, dual)
                with pytest.raises(RuntimeError, match="no gradient"):
                    route_experts(dual, 2)
    _lib.inference_only("this", x)
