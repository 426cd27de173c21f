"""Limits of the context operators that are checked before anything reaches a device (CPU only)."""
import pytest
import torch

from vidseg_diffusion_amd import _lib, ops
from vidseg_diffusion_amd._lib import VidsegError


@pytest.mark.parametrize("heads,kv_heads", [(131072, None), (1025, None), (2048, 2)])
def test_number_of_heads(heads, kv_heads):
    """More heads than the library takes are refused by their number: rows of 2^24 elements cannot be made any shorter by copying them."""
    q = torch.zeros(1, 1, heads * 128, dtype=torch.float16)
    k = q[..., :(kv_heads or heads) * 128]
    with pytest.raises(VidsegError, match="heads"):
        ops.cross_attention(q, k, k, heads, kv_heads=kv_heads)
    with pytest.raises(VidsegError, match="heads"):
        ops.prefix_attention(q, k[0], k[0], k, k, heads, kv_heads=kv_heads)


def test_rows_are_copied_once_at_most():
    from vidseg_diffusion_amd.context_ops import _heads_of
    rows = torch.zeros(1, 1, 1 << 24, dtype=torch.float16)                          # already contiguous, and as long as a stride may not be
    with pytest.raises(VidsegError, match="rows"):
        _heads_of(rows, 128)
    far = torch.zeros(1).to(torch.float16).as_strided((2, 1, 64), (0, 1 << 24, 0))
    t, _, b, n, h = _heads_of(far, 64)
    assert t.is_contiguous() and (b, n, h) == (64, 64, 64)


def test_forward_mode_derivatives_are_refused():
    """A dual tensor asks for no gradient, but a result without a tangent would read as a derivative of zero."""
    import torch.autograd.forward_ad as fwd
    x, g, b = torch.zeros(2, 4, 64), torch.ones(64), torch.zeros(64)
    q = torch.zeros(2, 3, 128, dtype=torch.float16)
    with fwd.dual_level():
        dual = lambda t: fwd.make_dual(t, torch.ones_like(t))                       # noqa: E731
        for a in ((dual(x), g, b), (x, dual(g), b), (x, g, dual(b))):
            with pytest.raises(VidsegError, match="forward-mode"):
                ops.groupnorm_act(*a, groups=8)
        for i in range(3):
            a = [dual(q) if j == i else q for j in range(3)]
            with pytest.raises(VidsegError, match="forward-mode"):
                ops.cross_attention(*a, 2)
        for i in range(5):
            a = [q, q[0], q[0], q, q]
            a[i] = dual(a[i])
            with pytest.raises(VidsegError, match="forward-mode"):
                ops.prefix_attention(*a, 2)
        with pytest.raises(VidsegError, match="HIP device"):                        # a level without dual operands changes nothing
            ops.cross_attention(q, q, q, 2)


@pytest.mark.parametrize("scale", [2.5e38, 3.0e38, 1e39, 1e-50])
def test_scales_that_fp32_cannot_hold(scale):
    """scale * log2 e is what the kernels multiply by: it has to be finite (0 * inf would be NaN), and the scale itself not zero in fp32."""
    p = 4096                                                                        # a pointer that is never followed
    for name, args in (("vidseg_context_attention_fwd", (p, 192, 64, 64, None, 0, 0, None, 0, 0, p, 320, 64, 64, p, 320, 64, 64, None, None, 0, p, None, None, 1, 1, 3, 0, 5,
                                                         1, 1, 64, scale, 0, None, 0, None)),
                       ("vidseg_context_attention_bwd", (*(p, 192, 64, 64) * 2, *(p, 320, 64, 64) * 2, None, None, 0, None, None, p, p, p, p, 1, 1, 1, 3, 5, 1, 1, 64, scale,
                                                         None, 0, None))):
        assert getattr(_lib.lib(), name)(*args) == -1, name
        assert b"scale" in _lib.lib().vidseg_last_error()


def test_row_numbers_stay_within_32_bits():
    """Row numbers are 32-bit, and the last tile of 128 runs past the last row: 2^31 - 8 rows (34 GB of queries, 8 wide) are refused."""
    for B, Nq, H in ((1, (1 << 28) - 1, 8), (1, (1 << 28) - 16, 8), (7, 1 << 28, 2)):
        assert _lib.lib().vidseg_context_attention_scratch_kib(B, Nq, 0, 5, H, 1, 8) == -1
        assert b"too many rows" in _lib.lib().vidseg_last_error()
    assert _lib.lib().vidseg_context_attention_scratch_kib(1, (1 << 28) - 64, 0, 5, 8, 1, 8) >= 0
    assert _lib.lib().vidseg_context_attention_bwd_scratch_kib(1, 1, (1 << 28) - 1, 5, 8, 1, 8) == -1
