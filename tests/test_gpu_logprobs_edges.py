"""Log probabilities at the ends of their range, against 64 bits, with the bounds of
test_gpu_logprobs.py."""

import math

import pytest
import torch

from oracle import step_oracle as O
from tests.test_gpu_logprobs import BF16, F32, check, inputs

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def in_fp32s_range(monkeypatch):
    """The 64-bit log probabilities as fp32 holds them: at small temperatures the type's lowest logit
    has one of -2e68, which is -inf there."""
    logprobs = O.logprobs

    def held(*args):
        lp, h, tlp, ids = logprobs(*args)
        return tuple(torch.where(v < torch.finfo(F32).min, -math.inf, v) for v in (lp, h, tlp)) + (ids,)
    monkeypatch.setattr(O, "logprobs", held)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("V", [70, 1003, 20001])
@pytest.mark.parametrize("temperature", [2.0 ** -99, 2.0 ** -60, 2.0 ** 40, 2.0 ** 66])
def test_temperatures_at_the_ends_of_the_range(temperature, V, dtype):
    """Powers of two, which fp32 holds as they are.  Masked places have no probability at any of
    them, nor have the places past a row's end."""
    x, tok = inputs(12, V, dtype, 3)
    x[1, V // 2:] = -math.inf
    tok[1] = 3
    x[2, 5:] = -math.inf
    tok[2] = V - 1
    x[3] = -math.inf
    x[4] = 1.5
    x[5, ::3] = torch.finfo(dtype).min
    check(x, tok, 0, temperature)
    check(x, tok, 5, temperature)
