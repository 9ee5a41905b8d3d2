"""Calls of the matching-transformer operators that their documentation allows or refuses beside the
ordinary ones: the operators under ``torch.ops.stereocv``, derivatives of other kinds, far values."""
import math

import pytest
import torch

from oracle import matching_oracle as O
from realtime_stereo_matcher_amd import functional as F
from realtime_stereo_matcher_amd import library  # noqa: F401  (registers the ops)

gpu = pytest.mark.gpu
ops = torch.ops.stereocv


class Reached(Exception):
    """Raised in place of a launch."""


@pytest.fixture
def no_launch(monkeypatch):
    """Host tensors pass for tensors of device 0, and a call that gets as far as the native library
    raises Reached: what the checks let through shows on the CPU."""
    def load():
        raise Reached

    def one_device(*ts):
        kinds = {t.device.type for t in ts}
        if kinds != {"cpu"}:
            raise RuntimeError(f"tensors on different devices: {kinds}")
        return 0

    monkeypatch.setattr(F, "_one_device", one_device)
    monkeypatch.setattr(F, "_device_check", one_device)
    monkeypatch.setattr(F._lib, "load", load)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)


# ------------------------------------------------------- the operators under torch.ops check as well
@pytest.mark.parametrize("inverse", [False, True])
@pytest.mark.parametrize("case", ["fine", "rank", "double", "short", "batch", "float positions", "frequencies",
                                  "rows of frequencies", "too many", "none", "layout", "device", "host"])
def test_rotary_op_refuses(case, inverse, request):
    """The turn back is checked as the turn is: before anything is read."""
    if case != "host":
        request.getfixturevalue("no_launch")
    x, p, f, layout, error = (torch.zeros(2, 3, 1, 8), torch.arange(3), F.rotary_frequencies(8), "half", RuntimeError)
    if case == "fine":
        error = Reached
    elif case == "rank":
        x = x[0]
    elif case == "double":
        x, error = x.double(), TypeError
    elif case == "short":
        p = torch.arange(2)
    elif case == "batch":
        p = torch.arange(9).view(3, 3)
    elif case == "float positions":
        p = p.float()
    elif case == "frequencies":
        f = f.float()
    elif case == "rows of frequencies":
        f = f[None]
    elif case == "too many":
        f = F.rotary_frequencies(10)
    elif case == "none":
        f = f[:0]
    elif case == "layout":
        layout, error = "halves", ValueError
    elif case == "device":
        f = f.to("meta")
    call = library._rot if case == "device" else ops.rotary  # (a meta tensor would select the fake kernel)
    with pytest.raises(error):
        call(x, p, f, layout, 1.0, inverse)
