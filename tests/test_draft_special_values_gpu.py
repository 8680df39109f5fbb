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
