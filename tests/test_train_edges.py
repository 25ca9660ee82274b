"""The training operators' refusals at the edges of what they take, on the CPU: no call
here reaches a launch."""
from __future__ import annotations

import pytest
import torch

from simple_llm_amd import _lib
from simple_llm_amd.gpu import gpu
from simple_llm_amd.gpu.gpu_pass_optimizer import _check_state
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


def _state(bits):
    kind = torch.float32 if bits == 32 else torch.uint8
    m, v = torch.zeros(256, dtype=kind), torch.zeros(256, dtype=kind)
    scales = [torch.zeros(2, dtype=torch.uint8) for _ in "mv"] if bits == 8 else [None, None]
    return gpu.AdamWState([torch.zeros(200)], [torch.zeros(200)], [torch.zeros(200).bfloat16()], bits,
                          [0], 3, m, v, *scales, torch.zeros(2, dtype=torch.int32),
                          torch.zeros(1, 6, dtype=torch.int64), torch.zeros(1, 2, dtype=torch.int32))


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_state_cannot_be_replaced(bits):
    """What the kernel reaches by its address, by assignment: a tensor of another type, size
    or device, or a count that the kernel would not see."""
    s = _state(bits)
    for name, other in (("m", torch.zeros(5)), ("v", torch.zeros(256, dtype=torch.float64)),
                        ("m_scale", torch.zeros(1)), ("v_scale", None), ("bits", 40 - bits),
                        ("step", torch.ones(1, dtype=torch.int32))):
        with pytest.raises(AttributeError):
            setattr(s, name, other)
    for seed in (-1, 1 << 32):
        with pytest.raises(ValueError, match="seed must"):
            s.seed = seed
    s.seed = 7
    assert s.seed == 7 and s.step.item() == 0


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_state_cannot_move(bits):
    """The same through a tensor's data, for every tensor that is held."""
    names = ["m", "v", "step"] + (["m_scale", "v_scale"] if bits == 8 else [])
    held = [lambda s, n=n: getattr(s, n) for n in names] + [
        lambda s, n=n: getattr(s, n)[0] for n in ("params", "grads", "copies")]
    for get in held:
        s = _state(bits)
        with pytest.raises(ValueError, match="the state lives on cpu"):  # the check behind it
            _check_state(_ctx(), s)
        at = get(s).data_ptr()
        get(s).data = torch.zeros(5)
        with pytest.raises(ValueError, match="no longer where it was"):
            _check_state(_ctx(), s)
        # and the memory is still the state's, whatever is allocated next
        assert at in [t.data_ptr() for t in s._memory]


def test_adamw_gradients_keep_their_type():
    """The lists are the program's own; the kernel's types are those of the making."""
    s = _state(32)
    s.grads[0] = torch.zeros(200).bfloat16()
    assert s._grad_dtype == torch.float32


def test_adamw_read_refuses_more_than_a_launch():
    """A lane for 8 elements, 256 a workgroup, fewer than 2^32 lanes: the last size that gets
    as far as the overlaps, and the next ones."""
    L = _lib.lib()
    most = 8 * ((1 << 32) - 256)
    for n, rc in ((most, _lib.SKV_E_INVALID), (most + 128, _lib.SKV_E_UNSUPPORTED),
                  (1 << 35, _lib.SKV_E_UNSUPPORTED), ((1 << 40) - 128, _lib.SKV_E_UNSUPPORTED),
                  ((1 << 63) - 128, _lib.SKV_E_UNSUPPORTED)):
        assert L.skv_adamw_read(FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, n, 0, None) == rc, n


def test_embedding_backward_refuses_more_than_its_last_launch():
    """The third launch has 512 lanes for 8 ranges of 16 tokens: it reaches 2^32 lanes before
    the second one does. The workspace's size is the last check before the overlaps."""
    L = _lib.lib()
    for T, d in ((1 << 30) - 128, 8), ((1 << 29) - 64, 257), (1 << 20, 250 * 256):
        units = -(-T // 16) * -(-d // 256)
        assert units <= (1 << 26) - 8
        need = L.skv_embedding_bwd_workspace_bytes(T, 10, d)
        assert L.skv_embedding_bwd(FAKE, FAKE, FAKE, T, 10, d, 1.0, 0, FAKE, need - 1, 0,
                                   None) == _lib.SKV_E_WORKSPACE
    for T, d in ((1 << 30) - 127, 8), ((1 << 30) - 64, 8), ((1 << 30) - 48, 8), (1 << 20, 1 << 18):
        assert L.skv_embedding_bwd(FAKE, FAKE, FAKE, T, 10, d, 1.0, 0, FAKE, 1 << 62, 0,
                                   None) == _lib.SKV_E_UNSUPPORTED, (T, d)
