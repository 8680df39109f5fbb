"""Bits that the drafted-decoding operators keep between their inputs and
their results."""

import numpy as np
import pytest

import draft_reference as ref

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import private_genomic_dnagpt_b200 as eng  # noqa: E402

from test_draft_gpu import HALF, f64, inputs, tree  # noqa: E402


@pytest.fixture(scope="module")
def cc():
    return eng.GenCryptoContext(eng.CCParams(ring_dim_log=10, limbs=3, dnum=1, seed=3))


# a softmax weight's half step between the two products
WEIGHT = {torch.bfloat16: 2.0 ** -16, torch.float16: 2.0 ** -22, torch.float32: 2.0 ** -24}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [(1, 1, 12, 12, 64, [103], 1), (2, 21, 4, 2, 64, [1000, 513], 2),
                                   (1, 33, 8, 4, 128, [2000], 3), (1, 5, 2, 2, 128, [3000], 1),
                                   (1, 64, 4, 2, 128, [900], 2), (1, 32, 4, 2, 64, [1500], 2),
                                   (1, 8, 2, 2, 256, [1000], 2), (1, 40, 2, 1, 192, [1200], 2),
                                   (2, 64, 4, 2, 256, [700, 64], 2)])
def test_attention_rounds_its_result_only(cc, dtype, shape):
    """An element is off by half a step of itself and, of sum p |v|, by a
    weight's half step and by the scores' and sums' roundings (the D + 8 and
    N + 8 terms at the top of test_draft_gpu)."""
    B, n, Hq, Hk, D, lens, branch = shape
    x = inputs(dtype, B, n, Hq, Hk, D, max(lens) + 3, lens, [tree(n, branch)] * B, seed=30)
    out, _ = cc.draft_attention(**x)
    want, _, mag, big, keys = ref.attention(*(f64(x[k]) for k in ("q", "k_cache", "v_cache")), lens, f64(x["k_new"]),
                                            f64(x["v_new"]), x["parents"].cpu().numpy(), D ** -0.5)
    noise = 2.0 ** -23 * ((D + 8) * big + keys + 8)
    room = HALF[dtype] * np.abs(want) + (WEIGHT[dtype] + noise)[..., None] * (1 + HALF[dtype]) * mag
    worst = (np.abs(f64(out) - want) / room).max()
    assert worst <= 1.0, f"{worst:.3g} times the bound"
