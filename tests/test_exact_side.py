"""The exact side of a decode step on the host: what its entry points refuse before anything is launched."""

import ctypes

import pytest
import torch

import cfm_b200  # noqa: F401
from cfm_b200 import _native
from cfm_b200.runtime.fidelity import compare_logits, token_logprobs
from cfm_b200.runtime.routed import RoutedExperts
from cfm_b200.runtime.routing import route_tokens
from cfm_b200.runtime.vllm_binding import BoundBlock

NULL, SHAPE, CAPACITY, UNSUPPORTED = -1, -2, -3, -4


@pytest.fixture(scope="module")
def library():
    if not _native.LIBRARY.exists():
        _native.build()
    return _native.load()


def rows(rows=2, columns=64, stride=None, kind=2, data=4096):
    return ctypes.byref(_native.Rows(data, columns if stride is None else stride, rows, columns, kind))


def test_struct_sizes_match_the_header():
    pointer = ctypes.sizeof(ctypes.c_void_p)
    assert ctypes.sizeof(_native.Rows) == pointer + 8 + 4 * 4
    assert ctypes.sizeof(_native.Experts) == 6 * 4 + 2 * pointer


def test_rows_that_the_entry_points_refuse(library):
    def route(x, top_k=4, out=4096):
        return library.cfm_route_tokens(x, top_k, 1, out, 0, out, 0, None)

    def scores(x, top=4, out=4096):
        return library.cfm_token_logprobs(x, out, 1, top, out, out, out, out, None)

    def compare(x, y=None, out=4096):
        return library.cfm_compare_logits(x, y or x, out, out, None)

    for call in (route, scores, compare):
        assert call(None) == NULL if call is not compare else library.cfm_compare_logits(None, None, 4096, 4096, None) == NULL
        assert call(rows(data=None)) == NULL
        assert call(rows(kind=3)) == UNSUPPORTED and call(rows(kind=-1)) == UNSUPPORTED
        assert call(rows(columns=0)) == SHAPE and call(rows(rows=-1)) == SHAPE
        assert call(rows(stride=63)) == SHAPE
        assert call(rows(data=4098)) == SHAPE  # FP32 off its alignment
        assert call(rows(rows=0)) == 0         # nothing to do
        assert call(rows(), out=None) == NULL
    assert route(rows(columns=1025)) == SHAPE
    for top_k in (0, 33, 65, -1):
        assert route(rows(), top_k) == SHAPE
    assert scores(rows(), -1) == SHAPE and scores(rows(), 33) == SHAPE and scores(rows(columns=3), 4) == SHAPE
    assert scores(rows(columns=(1 << 21) + 1)) == SHAPE
    for other in (rows(rows=3), rows(columns=63), rows(kind=0)):
        assert compare(rows(), other) == SHAPE


def test_layers_that_the_entry_points_refuse(library):
    def layer(hidden=256, width=48, experts=4, top_k=2, activation=0):
        return ctypes.byref(_native.Experts(hidden, width, experts, top_k, activation, 0, 4096, 4096))

    size = library.cfm_experts_workspace_bytes(layer(), 8)
    # Two BF16 terms of the activations and an FP32 row of every pair at least.
    assert size >= 8 * 2 * (48 * 4 + 256 * 4) and size % 256 == 0
    assert library.cfm_experts_workspace_bytes(layer(), 16) > size
    assert library.cfm_experts_workspace_bytes(None, 8) == NULL
    for bad in (dict(hidden=0), dict(hidden=250), dict(hidden=65664), dict(width=40), dict(width=0), dict(experts=0),
                dict(experts=4097), dict(top_k=0), dict(top_k=33)):
        assert library.cfm_experts_workspace_bytes(layer(**bad), 8) == SHAPE, bad
    assert library.cfm_experts_workspace_bytes(layer(activation=2), 8) == UNSUPPORTED
    for capacity in (0, -1, 1 << 23):
        assert library.cfm_experts_workspace_bytes(layer(), capacity) == CAPACITY

    def forward(tokens=4, workspace=4096, **changes):
        call = _native.Call(tokens, 0, 0, 0, 0, 0, 4096, 4096, 4096, None, 4096)
        for name, value in changes.items():
            setattr(call, name, value)
        return library.cfm_experts_forward(layer(), workspace, 8, ctypes.byref(call), None)

    assert forward(tokens=0) == CAPACITY and forward(tokens=9) == CAPACITY
    assert forward(workspace=None) == NULL
    for name in ("hidden", "ids", "weights", "out"):
        assert forward(**{name: None}) == NULL
    for name in ("hidden", "out"):
        assert forward(**{name: 4104}) == SHAPE  # off a 16-byte boundary
    assert library.cfm_experts_forward(layer(), 4096, 8, None, None) == NULL


def test_tensors_off_the_device_are_refused():
    x, tokens = torch.randn(2, 64), torch.zeros(2, dtype=torch.int64)
    for call in (lambda: route_tokens(x, 4), lambda: token_logprobs(x, tokens), lambda: compare_logits(x, x),
                 lambda: RoutedExperts(torch.zeros(2, 32, 128).bfloat16(), torch.zeros(2, 128, 16).bfloat16(), 1, 4)):
        with pytest.raises(ValueError):
            call()


def test_the_binding_knows_its_routers():
    with pytest.raises(ValueError, match="router"):
        BoundBlock(torch.nn.Linear(2, 2), None, 2, True, router="triton")
    logits = torch.randn(3, 16)
    weights, ids = BoundBlock(torch.nn.Linear(2, 2), None, 2, True).route(logits)
    assert torch.equal(ids.long(), logits.topk(2).indices)
