"""DraftModel's bookkeeping and EncryptedModel's tree of drafts, with the
operators and the encrypted blocks stood in for."""

from types import SimpleNamespace

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import private_genomic_dnagpt_b200 as eng  # noqa: E402
from private_genomic_dnagpt_b200 import drafting  # noqa: E402


@pytest.fixture
def operators(monkeypatch):
    """Operators that keep the lengths only; the cuts that were made."""
    cuts = []

    def attention(cc, q, k_cache, v_cache, lens, k, v, parents, scale=None):
        assert int(lens.max()) + q.shape[1] <= k_cache.shape[2]
        return torch.zeros_like(q), torch.zeros(q.shape[:3])

    def evict(cc, k, v, acc, lens, budget, recent, out=None):
        cuts.append(lens.tolist())
        return (*out, None, lens.clamp(max=budget))

    monkeypatch.setattr(drafting, "attention", attention)
    monkeypatch.setattr(drafting, "commit", lambda cc, k, v, lens, kn, vn, path, count: lens + count)
    monkeypatch.setattr(drafting, "accumulate", lambda *a: None)
    monkeypatch.setattr(drafting, "evict", evict)
    real = torch.device
    monkeypatch.setattr(torch, "device", lambda *a: real("cpu"))
    return cuts


def draft_model(capacity, budget, batch=1):
    w = dict(ln1=np.ones(8), ln2=np.ones(8), attn_qkv=np.zeros((24, 8)), attn_proj=np.zeros((8, 8)),
             mlp_fc=np.zeros((16, 8)), mlp_proj=np.zeros((8, 16)))
    cc = SimpleNamespace(params=SimpleNamespace(device=0))
    return drafting.DraftModel(cc, [w], capacity, batch=batch, heads=2, dtype=torch.float32, budget=budget, recent=8)


def step(m, nodes, counts):
    m.forward(torch.zeros(len(counts), nodes, 8), torch.full((len(counts), nodes), -1, dtype=torch.int32))
    m.accept(torch.zeros(len(counts), nodes, dtype=torch.int32), torch.tensor(counts, dtype=torch.int32))


def test_draft_model_cuts_when_a_tree_would_not_fit(operators):
    """Trees of 64 with one accepted node each: the cache is cut when its rows
    and the tree pass the capacity, not when the nodes offered so far do."""
    m = draft_model(300, 128)
    m.prefill(torch.zeros(1, 128, 8))
    for rows in range(128, 300 - 64 + 1):
        assert m.lens.tolist() == [rows] and not operators
        step(m, 64, [1])
    assert m.lens.tolist() == [237] and not operators
    step(m, 64, [1])
    assert operators == [[237]] and m.lens.tolist() == [129]


def test_draft_model_of_a_batch_cuts_for_its_longest_sequence(operators):
    m = draft_model(256, 150, batch=2)
    m.prefill(torch.zeros(2, 128, 8))
    for _ in range(5):
        step(m, 32, [16, 3])
    assert operators == [] and m.lens.tolist() == [208, 143]
    step(m, 32, [16, 3])
    assert operators == [] and m.lens.tolist() == [224, 146]
    step(m, 33, [1, 0])
    assert operators == [[224, 146]] and m.lens.tolist() == [151, 146]


def test_draft_model_without_a_budget_refuses(operators):
    m = draft_model(100, None)
    m.prefill(torch.zeros(1, 64, 8))
    for _ in range(10):
        step(m, 20, [1])
    with pytest.raises(ValueError, match="74 cached rows and 27 nodes"):
        step(m, 27, [1])


def test_a_refused_tree_leaves_no_block_with_drafts():
    """The second block refuses the tree: the first one is causal again."""
    class Block:
        def __init__(self, refuses):
            self.refuses, self.tree = refuses, ()

        def set_drafts(self, parents=(), first=None):
            if self.refuses and len(parents):
                raise eng.CKKSError(2, "the block's context was destroyed")
            self.tree = tuple(parents)

    model = eng.EncryptedModel.__new__(eng.EncryptedModel)
    model.blocks = [Block(False), Block(True)]
    with pytest.raises(eng.CKKSError):
        model.forward(np.zeros((4, 8)), [-1, 0])
    assert model.blocks[0].tree == ()
