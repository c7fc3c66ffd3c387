"""Requests at the limits of what they may bring, in captured decode steps."""
import pytest
import torch

from .test_request_limits_cpu import check_long_bias_lists, make_engine

pytestmark = pytest.mark.gpu


def test_bias_lists_up_to_the_limit_captured():
    check_long_bias_lists(make_engine("cuda", torch.bfloat16)[2])
