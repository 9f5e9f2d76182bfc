"""Routed experts on the CPU: what the C ABI and the operators refuse before any launch, and the sizes of workspaces."""
import pytest
import torch

from khaosz_amd import _abi, ops

P = 1 << 20  # a fake, aligned pointer: refused before any launch


def _route(**change):
    a = dict(logits=P, dtype=1, T=3, E=8, ld=8, k=2, renormalize=1, weights=P, experts=P, rows=P, tokens=P, offsets=P, ws=None, ws_bytes=0, stream=None)
    a.update(change)
    return _abi.load().aq_route_topk(*a.values())


@pytest.mark.parametrize("change,code", [
    (dict(dtype=2), -3), (dict(T=-1), -2), (dict(E=0), -2), (dict(k=0), -2), (dict(k=9), -2), (dict(ld=7), -2), (dict(E=513, ld=513), -6),
    (dict(E=64, ld=64, k=17), -6), (dict(T=(1 << 24) + 1), -6), (dict(logits=None), -1), (dict(weights=None), -1), (dict(experts=None), -1),
    (dict(rows=None), -1), (dict(tokens=None), -1), (dict(offsets=None), -1), (dict(logits=P + 1), -4), (dict(dtype=0, logits=P + 2), -4),
    (dict(weights=P + 2), -4), (dict(experts=P + 2), -4), (dict(rows=P + 2), -4), (dict(tokens=P + 2), -4), (dict(offsets=P + 2), -4),
    (dict(T=5000), -1), (dict(T=5000, ws=P), -5), (dict(T=5000, ws=P + 2, ws_bytes=1 << 20), -4),
])
def test_routing_is_refused_before_any_launch(change, code):
    assert _route(**change) == code


def _linear(**change):
    a = dict(xq=P, sx=P, x_rows=5, wq=P, sw=P, bias=None, bias_dtype=0, offsets=P, E=4, tokens=P, R=7, y=P, y_dtype=1, N=48, K=64, stream=None)
    a.update(change)
    return _abi.load().aq_linear_w8a8_grouped(*a.values())


GROUPED = [
    (dict(x_rows=-1), -2), (dict(E=0), -2), (dict(R=-1), -2), (dict(K=0), -2), (dict(K=24), -2), (dict(tokens=None), -2), (dict(E=513), -6),
    (dict(x_rows=1 << 27), -6), (dict(R=1 << 31), -6), (dict(xq=None), -1), (dict(sx=None), -1), (dict(wq=None), -1), (dict(sw=None), -1),
    (dict(offsets=None), -1), (dict(xq=P + 8), -4), (dict(wq=P + 8), -4), (dict(sx=P + 2), -4), (dict(sw=P + 2), -4), (dict(offsets=P + 2), -4),
    (dict(tokens=P + 2), -4), (dict(R=0), 0), (dict(K=1 << 27), -6),
]


@pytest.mark.parametrize("change,code", GROUPED + [(dict(y_dtype=2), -3), (dict(bias=P, bias_dtype=3), -3), (dict(N=0), -2), (dict(N=1 << 25), -6), (dict(y=None), -1),
                                                   (dict(y=P + 8), -4), (dict(bias=P + 2), -4)])
def test_grouped_linear_is_refused_before_any_launch(change, code):
    assert _linear(**change) == code


def _swiglu(**change):
    a = dict(xq=P, sx=P, x_rows=5, wq=P, sw=P, offsets=P, E=4, tokens=P, R=7, h=P, h_dtype=1, F=48, K=64, stream=None)
    a.update(change)
    return _abi.load().aq_swiglu_w8a8_grouped(*a.values())


@pytest.mark.parametrize("change,code", GROUPED + [(dict(h_dtype=2), -3), (dict(F=0), -2), (dict(F=40), -2), (dict(F=1 << 24), -6), (dict(h=None), -1), (dict(h=P + 8), -4)])
def test_grouped_swiglu_is_refused_before_any_launch(change, code):
    assert _swiglu(**change) == code


def _combine(**change):
    a = dict(y=P, dtype=1, R=6, N=16, rows=P, weights=P, T=3, k=2, residual=None, out=P, stream=None)
    a.update(change)
    return _abi.load().aq_combine_rows(*a.values())


@pytest.mark.parametrize("change,code", [
    (dict(dtype=2), -3), (dict(R=-1), -2), (dict(N=0), -2), (dict(T=-1), -2), (dict(k=0), -2), (dict(k=65), -6), (dict(N=(1 << 24) + 1), -6),
    (dict(T=(1 << 24) + 1), -6), (dict(R=1 << 31), -6), (dict(y=None), -1), (dict(rows=None), -1), (dict(weights=None), -1), (dict(out=None), -1),
    (dict(y=P + 1), -4), (dict(residual=P + 1), -4), (dict(out=P + 1), -4), (dict(rows=P + 2), -4), (dict(weights=P + 2), -4), (dict(T=0), 0),
])
def test_combination_is_refused_before_any_launch(change, code):
    assert _combine(**change) == code


def _experts(**change):
    a = dict(x=P, dtype=1, T=3, dim=64, offsets=P, E=4, tokens=P, rows=P, weights=P, k=2, up_gate=P, up_gate_scale=P, down=P, down_scale=P, F=32,
             residual=None, out=P, ws=P, ws_bytes=1 << 20, stream=None)
    a.update(change)
    return _abi.load().aq_experts_w8a8(*a.values())


@pytest.mark.parametrize("change,code", [
    (dict(dtype=2), -3), (dict(T=-1), -2), (dict(dim=0), -2), (dict(dim=40), -2), (dict(E=0), -2), (dict(k=0), -2), (dict(F=0), -2), (dict(F=24), -2),
    (dict(E=513), -6), (dict(k=65), -6), (dict(T=(1 << 24) + 1), -6), (dict(T=1 << 24, dim=256), -6), (dict(T=1 << 23, F=256), -6), (dict(dim=1 << 16, F=1 << 16), -6),
    (dict(x=None), -1), (dict(offsets=None), -1), (dict(tokens=None), -1), (dict(rows=None), -1), (dict(weights=None), -1), (dict(up_gate=None), -1),
    (dict(up_gate_scale=None), -1), (dict(down=None), -1), (dict(down_scale=None), -1), (dict(out=None), -1), (dict(ws=None), -1), (dict(x=P + 8), -4),
    (dict(up_gate=P + 8), -4), (dict(down=P + 8), -4), (dict(out=P + 8), -4), (dict(ws=P + 8), -4), (dict(offsets=P + 2), -4), (dict(tokens=P + 2), -4),
    (dict(rows=P + 2), -4), (dict(weights=P + 2), -4), (dict(up_gate_scale=P + 2), -4), (dict(down_scale=P + 2), -4), (dict(ws_bytes=100), -5), (dict(T=0), 0),
])
def test_experts_are_refused_before_any_launch(change, code):
    assert _experts(**change) == code


def test_sizes_of_workspaces():
    lib = _abi.load()
    assert lib.aq_route_topk_workspace_bytes(0, 8) == 0 and lib.aq_route_topk_workspace_bytes(1, 8) == 0
    assert lib.aq_route_topk_workspace_bytes((1 << 24) + 1, 8) == 0 and lib.aq_route_topk_workspace_bytes(5000, 0) == 0
    assert lib.aq_route_topk_workspace_bytes(1 << 24, 512) <= 513 * 512 * 6  # larger batches: larger chunks
    size = lib.aq_experts_w8a8_workspace_bytes
    assert size(1, 0, 2, 64, 32) == 0 and size(1, 3, 0, 64, 32) == 0 and size(1, 3, 65, 64, 32) == 0
    assert size(0, 100, 2, 64, 32) > size(1, 100, 2, 64, 32) >= 100 * 64 + 200 * 32 + 200 * 64 * 2


def test_cpu_tensors_are_refused():
    x, logits = torch.zeros(3, 64), torch.zeros(3, 4)
    rows = torch.zeros(3, 2, dtype=torch.int32)
    codes, scales = torch.zeros(4, 64, 64, dtype=torch.int8), torch.ones(4, 64)
    offsets = torch.zeros(5, dtype=torch.int32)
    r = ops.Routing(torch.ones(3, 2), rows, rows, torch.zeros(6, dtype=torch.int32), offsets)
    for call in (lambda: ops.route_topk(logits, 2),
                 lambda: ops.linear_w8a8_grouped(torch.zeros(3, 64, dtype=torch.int8), torch.ones(3), codes, scales, offsets),
                 lambda: ops.swiglu_w8a8_grouped(torch.zeros(3, 64, dtype=torch.int8), torch.ones(3), codes, scales, offsets),
                 lambda: ops.combine_rows(x, rows, torch.ones(3, 2)),
                 lambda: ops.experts_w8a8(x, r, codes, scales, torch.zeros(4, 64, 32, dtype=torch.int8), scales)):
        with pytest.raises(RuntimeError):
            call()
