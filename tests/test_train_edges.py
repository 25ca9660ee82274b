"""The training operators' refusals at the edges of what they take, on the CPU: no call
here reaches a launch."""
from __future__ import annotations

import pytest

from simple_llm_amd import _lib
from simple_llm_amd.gpu import gpu
from test_train import FAKE, _ctx


@pytest.mark.parametrize("eps", [1e-40, 2.0 ** -127, -1e-8, float("nan")])
def test_adamw_refuses_a_subnormal_eps(eps):
    """The hardware takes it for 0, and 0 / eps would be a NaN and not 0."""
    with pytest.raises(ValueError, match="eps must be 0, or at least"):
        gpu.adamw_update(_ctx(), None, 1e-3, eps=eps)
    L = _lib.lib()
    rc = L.skv_adamw(FAKE, FAKE, 3, FAKE, FAKE, None, None, FAKE, 32, 0, 1e-3, None, 0.9, 0.999, eps,
                     0.1, 1.0, None, 0, None)
    assert rc == _lib.SKV_E_INVALID and b"eps" in L.skv_last_error()
