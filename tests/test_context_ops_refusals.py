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


def _attn(**change):
    z = lambda *s: torch.zeros(*s, dtype=torch.float16)                            # noqa: E731
    a = dict(q=z(2, 3, 128), k=z(2, 5, 128), v=z(2, 5, 128), heads=2, kv_heads=None, k_lens=None, scale=None)
    a.update(change)
    return a


ATTN_REFUSED = [
    (dict(), "HIP device"),
    (dict(q=torch.zeros(2, 3, 128)), "float32"),
    (dict(q=torch.zeros(3, 128, dtype=torch.float16)), r"\[B, Nq"),
    (dict(heads=3), "heads"),
    (dict(heads=0), "heads"),
    (dict(kv_heads=4), "key heads"),
    (dict(kv_heads=0), "key heads"),
    (dict(heads=32), "head width 4"),
    (dict(q=torch.zeros(2, 3, 272, dtype=torch.float16), k=torch.zeros(2, 5, 272, dtype=torch.float16), v=torch.zeros(2, 5, 272, dtype=torch.float16)), "head width 136"),
    (dict(k=torch.zeros(2, 5, 128, dtype=torch.bfloat16)), "bfloat16"),
    (dict(k=torch.zeros(2, 5, 64, dtype=torch.float16)), "rows of 2 heads"),
    (dict(k=torch.zeros(3, 5, 128, dtype=torch.float16)), "samples"),
    (dict(v=torch.zeros(2, 6, 128, dtype=torch.float16)), "shape"),
    (dict(k_lens=torch.tensor([1, 2])), "k_lens"),
    (dict(k_lens=torch.tensor([1], dtype=torch.int32)), "k_lens"),
    (dict(scale=0.0), "scale"),
    (dict(scale=float("inf")), "scale"),
    (dict(scale=float("nan")), "scale"),
]


@pytest.mark.parametrize("change,word", ATTN_REFUSED + [
    (dict(key_mask=torch.ones(2, 5)), "key_mask"),
    (dict(key_mask=torch.ones(2, 4, dtype=torch.bool)), "key_mask"),
    (dict(key_mask=torch.ones(5, 2, dtype=torch.bool).t()), "key_mask"),
])
def test_cross_attention_refuses(change, word):
    a = _attn(**change)
    with pytest.raises(VidsegError, match=word):
        ops.cross_attention(a.pop("q"), a.pop("k"), a.pop("v"), a.pop("heads"), **a)


@pytest.mark.parametrize("change,word", ATTN_REFUSED + [
    (dict(k_prefix=torch.zeros(7, 64, dtype=torch.float16)), "k_prefix"),
    (dict(k_prefix=torch.zeros(2, 7, 128, dtype=torch.float16)), "k_prefix"),
    (dict(k_prefix=torch.zeros(6, 128, dtype=torch.float16)), "prefix of 6"),
    (dict(k=torch.zeros(1, 5, 128, dtype=torch.float16), v=torch.zeros(1, 5, 128, dtype=torch.float16)), "samples"),
    (dict(q=torch.zeros(2, 3, 128, dtype=torch.float16, requires_grad=True)), "gradients"),
])
def test_prefix_attention_refuses(change, word):
    a = _attn(k_prefix=torch.zeros(7, 128, dtype=torch.float16), v_prefix=torch.zeros(7, 128, dtype=torch.float16))
    a.update(change)
    if a["q"].dtype == torch.float16 and a["q"].shape[-1] == 272:
        a["k_prefix"] = a["v_prefix"] = torch.zeros(7, 272, dtype=torch.float16)
    with pytest.raises(VidsegError, match=word):
        ops.prefix_attention(a.pop("q"), a.pop("k_prefix"), a.pop("v_prefix"), a.pop("k"), a.pop("v"), a.pop("heads"), **a)


def test_context_attention_c_entry_refuses():
    from vidseg_diffusion_amd import _lib
    p = 4096

    def fwd(**k):
        a = dict(q=p, qb=192, qn=64, qh=64, kp=None, kpn=0, kph=0, vp=None, vpn=0, vph=0, k=p, kb=320, kn=64, kh=64, v=p, vb=320, vn=64, vh=64, lens=None,
                 mask=None, mb=0, out=p, lo=None, lse=None, dtype=1, B=1, Nq=3, Np=0, Nk=5, H=1, Hk=1, d=64, scale=0.125, causal=0, scratch=None, kib=0)
        a.update(k)
        return _lib.lib().vidseg_context_attention_fwd(*a.values(), None)
    for k in (dict(q=None), dict(out=None), dict(k=None), dict(Np=4), dict(dtype=0), dict(dtype=3), dict(B=0), dict(Nq=0), dict(Nk=-1), dict(H=3, Hk=2), dict(d=12), dict(d=136),
              dict(scale=0.0), dict(scale=float("nan")), dict(q=p + 2), dict(kn=63), dict(vh=4), dict(causal=1, mask=p), dict(Nq=1, Nk=4096), dict(B=60000, Nq=1 << 20)):
        assert fwd(**k) == -1, k
        assert b"context_attention" in _lib.lib().vidseg_last_error()
