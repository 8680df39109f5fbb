"""What the torch binding of the drafted-decoding operators refuses because
the C entry points would not see it."""

import pytest

torch = pytest.importorskip("torch")

from private_genomic_dnagpt_b200 import drafting  # noqa: E402

from test_draft_cpu import OPS, Reached, args, cc  # noqa: E402, F401


def test_sizes_past_32_bits(cc):  # noqa: F811
    """A capacity that 32 bits would cut to 10 is refused, not cut."""
    a = args("attention")
    with Reached():
        drafting.attention(cc, **a)
    for name in ("k_cache", "v_cache"):
        a[name] = a[name][:, :, :1].expand(2, 2, 2 ** 32 + 10, 8)
    with pytest.raises(ValueError, match="capacity: 4294967306"):
        drafting.attention(cc, **a)


@pytest.mark.parametrize("op", OPS)
def test_forward_mode_gradients_are_refused(cc, op):  # noqa: F811
    """A tangent would be dropped without a word, also under no_grad."""
    import torch.autograd.forward_ad as fwd
    for name, t in args(op).items():
        if isinstance(t, torch.Tensor) and t.is_floating_point():
            with fwd.dual_level(), torch.no_grad():
                a = args(op) | {name: fwd.make_dual(t, torch.ones_like(t))}
                with pytest.raises(ValueError, match="forward-mode"):
                    getattr(drafting, op)(cc, **a)
                with fwd._set_fwd_grad_enabled(False), Reached():
                    getattr(drafting, op)(cc, **a)


@pytest.mark.parametrize("op", OPS)
def test_negated_views_are_refused(cc, op):  # noqa: F811
    """The imaginary part of a conjugate is such a view."""
    assert torch.zeros(3, dtype=torch.complex64).conj().imag.is_neg()
    for name, t in args(op).items():
        if isinstance(t, torch.Tensor) and t.is_floating_point():
            with pytest.raises(ValueError, match="negated"):
                getattr(drafting, op)(cc, **(args(op) | {name: torch._neg_view(t)}))
