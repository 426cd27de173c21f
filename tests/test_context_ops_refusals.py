"""Calls that the context operators refuse, before anything reaches a device (CPU only)."""
import pytest
import torch

from vidseg_diffusion_amd import ops
from vidseg_diffusion_amd._lib import VidsegError


@pytest.mark.parametrize("change,word", [
    (dict(), "HIP device"),                                                       # CPU tensors: there is no CPU path
    (dict(x=torch.zeros(2, 4, 64, dtype=torch.float64)), "float64"),
    (dict(x=torch.zeros(64)), "[B, ..., C]"),
    (dict(groups=7), "groups"),
    (dict(groups=0), "groups"),
    (dict(act=2), "act"),
    (dict(eps=-1.0), "eps"),
    (dict(gamma=torch.ones(64, dtype=torch.float16)), "gamma"),
    (dict(gamma=torch.ones(32)), "gamma"),
    (dict(beta=torch.ones(1, 64)), "beta"),
    (dict(x=torch.zeros(1, 1, 8200), gamma=torch.ones(8200), beta=torch.ones(8200), groups=8), "8192"),
    (dict(x=torch.zeros(65536, 1, 64)), "65535"),
])
def test_groupnorm_act_refuses(change, word):
    a = dict(x=torch.zeros(2, 4, 64), gamma=torch.ones(64), beta=torch.zeros(64), groups=8, eps=1e-5, act=ops.ACT_SILU)
    a.update(change)
    with pytest.raises(VidsegError, match=word.replace("[", r"\[").replace("]", r"\]").replace(".", r"\.")):
        ops.groupnorm_act(a["x"], a["gamma"], a["beta"], groups=a["groups"], eps=a["eps"], act=a["act"])


def test_groupnorm_act_c_entry_refuses():
    """The C entry points check sizes and scratch themselves and return an error with a message; nothing is launched."""
    from vidseg_diffusion_amd import _lib
    p = 4096                                                                       # a pointer that is never followed

    def fwd(**k):
        a = dict(x=p, xb=256, xr=64, dtype=1, B=1, HW=4, C=64, G=8, gamma=p, beta=p, eps=1e-5, act=1, rows=4, y=p, mean=None, rstd=None, scratch=p, floats=16)
        a.update(k)
        return _lib.lib().vidseg_groupnorm_act_fwd(*a.values(), None)
    for k in (dict(x=None), dict(dtype=3), dict(C=65), dict(G=0), dict(xr=63), dict(act=2), dict(rows=0), dict(floats=15), dict(mean=p), dict(B=0), dict(HW=0)):
        assert fwd(**k) == -1, k
        assert b"groupnorm_act" in _lib.lib().vidseg_last_error()
