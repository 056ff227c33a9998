"""The largest finite numbers are finite numbers: arguments of the stand-alone operators at the ends of their ranges.
No GPU is needed: without rows nothing is launched."""
import pytest
import torch

from gpt_oss_amd_b200 import capi

LARGEST = torch.finfo(torch.float32).max


def _norm(eps):
    a = [0, 64, 0, 0, 64, 0, 0, 0, 0, 0, 0, 0, eps, 0, 0, 0, 0, 0, 0, 0]
    return capi.lib().moe_b200_add_rmsnorm(capi.packer(capi.AddRmsnormArgs)(*a), None)


def _route(scale):
    a = [0, 64, 4, 0, 0, 64, 0, 0, 1, 1, 1, 1, scale, 0, 0, 0]
    return capi.lib().moe_b200_route_logits(capi.packer(capi.RouteLogitsArgs)(*a), None)


@pytest.mark.parametrize("v,norm,route", [
    (0.0, True, True), (LARGEST, True, True), (3.2e38, True, True), (-LARGEST, False, True), (-1e-45, False, True),
    (float("inf"), False, False), (float("-inf"), False, False), (float("nan"), False, False)])
def test_finite_numbers(v, norm, route):
    assert _norm(v) == (capi.OK if norm else capi.ERR_INVALID)
    assert _route(v) == (capi.OK if route else capi.ERR_INVALID)
