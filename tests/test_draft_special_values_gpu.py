"""Infinities and NaN in the operands of the drafted-decoding operators, where
they count and where they do not."""

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import private_genomic_dnagpt_b200 as eng  # noqa: E402

from test_draft_gpu import TYPES, f64, i32, inputs, tree  # noqa: E402


@pytest.fixture(scope="module")
def cc():
    return eng.GenCryptoContext(eng.CCParams(ring_dim_log=10, limbs=3, dnum=1, seed=3))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [33, 64, 128, 200])
@pytest.mark.parametrize("nodes,heads", [(7, 1), (20, 2), (64, 2)])
@pytest.mark.parametrize("keys", [0, 90, 5000])
def test_values_that_are_not_finite_show_whatever_their_weight(cc, dtype, D, nodes, heads, keys):
    """A value that a row sees spoils its element of the row also where its
    weight is exp(-1000) of the others', on every kernel and wherever the list
    of keys is cut; it spoils nothing else."""
    parents = tree(nodes, 2)
    x = inputs(dtype, 1, nodes, heads, 1, D, max(keys, 1), [keys], [parents], seed=40)
    for name in ("q", "k_cache", "k_new"):
        x[name][..., 0] = 0.0
    x["q"][..., 0] = D ** 0.5
    clean = f64(cc.draft_attention(**x)[0])
    for at in [a for a in (0, 77, 2500, keys - 1) if 0 <= a < keys]:
        y = {k: v.clone() for k, v in x.items()}
        y["k_cache"][:, :, at, 0] = -1000.0
        y["v_cache"][:, :, at, 3] = float("inf")
        got = f64(cc.draft_attention(**y)[0])
        assert not np.isfinite(got[..., 3]).any(), at
        assert np.isfinite(np.delete(got, 3, -1)).all(), at
    # node 1's value, seen by node 1 and what hangs below it
    below = {1}
    for i, p in enumerate(parents):
        below |= {i} if p in below else set()
    x["k_new"][:, 1, :, 0] = -1000.0
    x["v_new"][:, 1, :, 2] = float("nan")
    got = f64(cc.draft_attention(**x)[0])
    for i in range(nodes):
        if i in below:
            # node 1 has no other key where the cache is empty
            assert not np.isfinite(got[:, i, :, 2]).any() and np.isfinite(np.delete(got[:, i], 2, -1)).all(), i
        else:
            assert np.array_equal(got[:, i], clean[:, i]), i


def accumulate_inputs(dtype, D, cap, length, heads=4, nodes=3, seed=41):
    x = inputs(dtype, 1, nodes, heads, 2, D, cap, [length], [tree(nodes, 1)], seed=seed)
    path, count = i32([list(range(nodes))]), i32([nodes])
    return x, path, count, torch.rand(1, 2, cap, device="cuda")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [33, 64, 128, 256])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_infinite_keys_get_no_weight(cc, dtype, D, sign):
    """A key whose score is -inf adds 0 to its weight, whatever bits the
    query's element has; the others' weights are what they were without it."""
    import draft_reference as ref
    x, path, count, acc = accumulate_inputs(dtype, D, 300, 290)
    x["q"][..., 5] = sign * torch.tensor([1.0, 0.75, 2.0, 1.0 / 3.0], device="cuda").to(dtype)
    x["k_cache"][:, :, [3, 150, 289], 5] = -sign * float("inf")
    _, lse = cc.draft_attention(**x)
    assert torch.isfinite(lse).all()
    cc.draft_commit(x["k_cache"], x["v_cache"], x["lens"], x["k_new"], x["v_new"], path, count)
    before = f64(acc)
    want = ref.accumulate(f64(x["q"]), f64(lse), f64(x["k_cache"]), [290], path.cpu().numpy(), [3], before, D ** -0.5)
    got = f64(cc.draft_accumulate(x["q"], lse, x["k_cache"], x["lens"], path, count, acc))
    assert np.array_equal(got[:, :, [3, 150, 289]], before[:, :, [3, 150, 289]])
    assert np.isfinite(got).all() and np.abs(got - want).max() <= 1e-3 * np.abs(want).max()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [33, 64])
def test_a_key_that_is_no_number_spoils_its_own_weight(cc, dtype, D):
    x, path, count, acc = accumulate_inputs(dtype, D, 300, 290)
    _, lse = cc.draft_attention(**x)
    want = f64(cc.draft_accumulate(x["q"], lse, x["k_cache"], x["lens"], path, count, acc.clone()))
    x["k_cache"][:, :, 77, D - 1] = float("nan")
    x["k_cache"][:, :, 293:] = float("nan")  # behind the last key
    got = f64(cc.draft_accumulate(x["q"], lse, x["k_cache"], x["lens"], path, count, acc))
    assert np.isnan(got[:, :, 77]).all()
    assert np.array_equal(np.delete(got, 77, 2), np.delete(want, 77, 2))


def test_largest_float32_keys(cc):
    """Elements next to the largest float32 number, with scores near 1."""
    x, path, count, acc = accumulate_inputs(torch.float32, 64, 300, 290)
    x["q"].fill_(2.0 ** -131)  # a denormal number
    x["k_cache"].fill_(0.0)
    x["k_cache"][:, :, ::2, 7] = 3.4e38
    acc.zero_()
    lse = torch.zeros(1, 3, 4, device="cuda")
    got = f64(cc.draft_accumulate(x["q"], lse, x["k_cache"], x["lens"], path, count, acc, 1.0))
    even = 6.0 * np.exp(float(np.float32(3.4e38)) * 2.0 ** -131)
    assert np.abs(got[0, :, 0:288:2] - even).max() <= 1e-5 * even
    assert np.abs(got[0, :, 1:288:2] - 6.0).max() <= 6e-5


def test_weights_that_are_no_numbers_are_evicted_first(cc):
    """The order of eviction by hand: numbers, then -inf, then NaN."""
    acc = torch.tensor([[[float("nan"), float("-inf"), -1.0, float("nan"), float("inf")]]], device="cuda")
    k = torch.arange(5.0, device="cuda")[None, None, :, None].clone()
    for budget, rows in ((1, [4]), (2, [2, 4]), (3, [1, 2, 4]), (4, [0, 1, 2, 4]), (5, [0, 1, 2, 3, 4])):
        got = cc.draft_evict(k, k.clone(), acc, i32([5]), budget, 0)
        assert got[3][0, 0].tolist() == rows and got[0][0, 0, :, 0].tolist() == rows
