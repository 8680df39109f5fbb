"""Bits that the drafted-decoding operators keep between their inputs and
their results."""

import numpy as np
import pytest

import draft_reference as ref

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import private_genomic_dnagpt_b200 as eng  # noqa: E402

from test_draft_gpu import HALF, f64, i32, inputs, tree  # noqa: E402


@pytest.fixture(scope="module")
def cc():
    return eng.GenCryptoContext(eng.CCParams(ring_dim_log=10, limbs=3, dnum=1, seed=3))


# a softmax weight's half step between the two products
WEIGHT = {torch.bfloat16: 2.0 ** -16, torch.float16: 2.0 ** -22, torch.float32: 2.0 ** -24}


@pytest.mark.parametrize("dtype", list(WEIGHT))
@pytest.mark.parametrize("shape", [(1, 1, 12, 12, 64, [103], 1), (2, 21, 4, 2, 64, [1000, 513], 2),
                                   (1, 33, 8, 4, 128, [2000], 3), (1, 5, 2, 2, 128, [3000], 1),
                                   (1, 64, 4, 2, 128, [900], 2), (1, 32, 4, 2, 64, [1500], 2),
                                   (1, 8, 2, 2, 256, [1000], 2), (1, 40, 2, 1, 192, [1200], 2),
                                   (2, 64, 4, 2, 256, [700, 64], 2)])
def test_attention_rounds_its_result_only(cc, dtype, shape):
    """An element is off by half a step of itself and, of sum p |v|, by a
    weight's half step and by the scores' and sums' roundings (the D + 8 and
    N + 8 terms at the top of test_draft_gpu).  In float16 a weight is the sum
    of two multiples of 2^-24 and the largest is 2^7 or more, so each is off by
    2^-31 of the row's sum at most, and results end at multiples of 2^-24."""
    B, n, Hq, Hk, D, lens, branch = shape
    x = inputs(dtype, B, n, Hq, Hk, D, max(lens) + 3, lens, [tree(n, branch)] * B, seed=30)
    out, _ = cc.draft_attention(**x)
    want, _, mag, big, keys = ref.attention(*(f64(x[k]) for k in ("q", "k_cache", "v_cache")), lens, f64(x["k_new"]),
                                            f64(x["v_new"]), x["parents"].cpu().numpy(), D ** -0.5)
    noise = 2.0 ** -23 * ((D + 8) * big + keys + 8)
    room = HALF[dtype] * np.abs(want) + (WEIGHT[dtype] + noise)[..., None] * (1 + HALF[dtype]) * mag
    if dtype == torch.float16:
        values = np.abs(np.concatenate([f64(x["v_cache"]), f64(x["v_new"]).swapaxes(1, 2)], 2)).sum(2)  # [B, Hk, D]
        room += 2.0 ** -31 * values[:, None].repeat(Hq // Hk, 2) + 2.0 ** -25
    worst = (np.abs(f64(out) - want) / room).max()
    assert worst <= 1.0, f"{worst:.3g} times the bound"


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("nodes", [1, 40, 128])
@pytest.mark.parametrize("ahead", [12.3, 14.0, 16.9, 17.6])
def test_attention_beside_a_heavy_key(cc, D, nodes, ahead):
    """float16: the first key's score is `ahead` above all others', its value
    is 0, so the result is made of weights of exp(-ahead) alone; the others'
    values are positive.  The bound is that of the test above, whose 2^-31 is
    the larger part here."""
    N, heads = 4000, 2 if nodes > 64 else 1
    nodes //= heads
    x = inputs(torch.float16, 1, nodes, heads, 1, D, N, [N], [tree(nodes, 2)], seed=31)
    for name in ("q", "k_cache", "k_new"):
        x[name].zero_()
    x["q"][..., 0] = D ** 0.5
    x["k_cache"][:, :, 0, 0] = ahead
    for name in ("v_cache", "v_new"):
        x[name].abs_().add_(0.25)
    x["v_cache"][:, :, 0] = 0.0
    out, lse = cc.draft_attention(**x)
    want, wlse, mag, big, keys = ref.attention(*(f64(x[k]) for k in ("q", "k_cache", "v_cache")), [N], f64(x["k_new"]),
                                               f64(x["v_new"]), x["parents"].cpu().numpy(), D ** -0.5)
    noise = 2.0 ** -23 * ((D + 8) * big + keys + 8)
    values = f64(x["v_cache"]).sum(2) + f64(x["v_new"]).sum(1)
    room = 2.0 ** -11 * np.abs(want) + (2.0 ** -22 + noise)[..., None] * (1 + 2.0 ** -11) * mag
    room += 2.0 ** -31 * values[:, None] + 2.0 ** -25
    assert (np.abs(f64(out) - want) / room).max() <= 1.0
    assert (np.abs(f64(lse) - wlse) <= 0.5 * noise + 2.0 ** -22 * (1 + np.abs(wlse))).all()


@pytest.mark.parametrize("D", [4, 8, 16])
def test_float32_weights_take_whole_products(cc, D):
    """Every element is 1 + 2^-11 - 2^-22 times a power of two, whose square
    lies 2^-22 of itself above what elements cut to twice 11 bits give without
    the product of their second parts.  With scale 1 the score S is off by two
    roundings of 2^-24 and the log-sum times log2(e) by one, ex2 by 2^-21 of
    the weight: the weight is off by 3 2^-24 S + 2^-21 of itself."""
    x = inputs(torch.float32, 1, 1, 1, 1, D, 200, [190], [[-1]], seed=32)
    v = 1 + 2.0 ** -11 - 2.0 ** -22
    x["q"].fill_(v * 1024 / D)
    x["k_cache"].fill_(v)
    S = D * float(x["q"][0, 0, 0, 0]) * float(x["k_cache"][0, 0, 0, 0])
    lse = torch.full((1, 1, 1), S, device="cuda")
    want = np.exp(S - float(lse[0, 0, 0]))
    got = f64(cc.draft_accumulate(x["q"], lse, x["k_cache"], x["lens"], i32([[0]]), i32([1]),
                                  torch.zeros(1, 1, 200, device="cuda"), 1.0))[0, 0, :191]
    assert np.abs(got - want).max() <= (3 * 2.0 ** -24 * S + 2.0 ** -21) * want
