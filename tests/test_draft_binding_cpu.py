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
