"""A workspace that is given as a buffer has its own size, which the library checks (on the CPU:
arguments are checked before anything else, and a call without a context names the first wrong one)."""
from types import SimpleNamespace

import pytest
import torch

import gotransformers_amd as gt

P = 1 << 40  # addresses that are only compared
X, Y, Z, U, V, W, A, B, D = (P + (i << 36) for i in range(9))


class NoContext(SimpleNamespace):
    handle = None

    def check(self, code):
        gt._check(code)


NORM = gt.norm_desc(gt.VALUES_BFLOAT16, 100, 2048)
BIAS = gt.grouped_desc(gt.VALUES_BFLOAT16, 4, 300, 64, 128)
ROUTE = gt.route_desc(gt.VALUES_FLOAT32, 1000, 64, 6)
ADAPTED = gt.adapted_desc(gt.VALUES_BFLOAT16, 50, 64, 128, 4, 8)
CALLS = {
    "norm_gradient": (gt.norm_workspace_bytes(NORM),
                      lambda c, *ws: gt.norm_gradient(c, NORM, X, Y, W, None, Z, A, gt.VALUES_FLOAT32, False, *ws)),
    "grouped_bias_gradient": (gt.grouped_bias_workspace_bytes(BIAS),
                              lambda c, *ws: gt.grouped_bias_gradient(c, BIAS, U, X, Y, gt.VALUES_FLOAT32, False, *ws)),
    "route_forward": (gt.route_workspace_bytes(ROUTE), lambda c, *ws: gt.route_forward(c, ROUTE, X, None, Y, Z, U, V, W, *ws)),
    "adapted_forward": (gt.adapted_workspace_bytes(ADAPTED), lambda c, *ws: gt.adapted_forward(c, ADAPTED, X, W, None, A, D, U, V, Y, *ws)),
}


@pytest.mark.parametrize("name", list(CALLS))
def test_workspaces_that_are_too_small(name):
    need, call = CALLS[name]
    whole = torch.empty(need + 64, dtype=torch.uint8)
    start = -whole.data_ptr() % 16
    buffer = whole[start:start + need]
    fine, small = "context is null", f"but the call needs {need}"
    for args, text in (((buffer,), fine), ((buffer[:need - 1],), small), ((whole[start:],), fine),
                       ((buffer, None, need - 1), small), ((buffer[:need - 1], None, need), small),
                       ((buffer.data_ptr(), None, need), fine), ((buffer.data_ptr(), None, need - 1), small),
                       ((buffer.data_ptr(),), fine), ((None,), "workspace")):
        with pytest.raises(gt.InvalidArgument, match=text):
            call(NoContext(), *args)


def test_a_buffer_of_wider_values_has_all_of_its_bytes():
    need, call = CALLS["route_forward"]
    buffer = torch.empty(-(-need // 8) + 8, dtype=torch.float64)
    assert buffer.data_ptr() % 16 == 0
    with pytest.raises(gt.InvalidArgument, match="context is null"):
        call(NoContext(), buffer)
