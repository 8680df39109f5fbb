"""DraftModel's packed prompts and 4-bit caches: the bookkeeping, with the
operators stood in for."""

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from private_genomic_dnagpt_b200 import drafting  # noqa: E402

from test_draft_model_cpu import draft_model, operators, step  # noqa: E402, F401


@pytest.fixture
def more(operators, monkeypatch):  # noqa: F811
    """Which of the operators were called, in their order."""
    calls = []

    def attention(name, cc, q, k_cache, v_cache, lens, k, v, parents, scale=None):
        calls.append(name)
        return torch.zeros_like(q), torch.zeros(q.shape[:3])

    def prompt(cc, q, k, v, starts, scale=None):
        calls.append("prompt")
        return torch.zeros_like(q), torch.zeros(q.shape[:2])

    def fill(name, cc, k_cache, v_cache, lens, k, v, starts):
        calls.append((name, k_cache.dtype, k_cache.shape[3]))
        return lens + starts[1:] - starts[:-1]

    def commit(name, cc, k, v, lens, kn, vn, path, count):
        calls.append(name)
        return lens + count

    monkeypatch.setattr(drafting, "prompt", prompt)
    for name in ("attention", "attention4"):
        monkeypatch.setattr(drafting, name, lambda *a, name=name: attention(name, *a))
    for name in ("commit", "commit4"):
        monkeypatch.setattr(drafting, name, lambda *a, name=name: commit(name, *a))
    for name in ("fill", "fill4"):
        monkeypatch.setattr(drafting, name, lambda *a, name=name: fill(name, *a))
    monkeypatch.setattr(drafting, "row4_bytes", lambda d: 12)
    return calls


def model(capacity, batch=1, **more):
    w = dict(ln1=np.ones(8), ln2=np.ones(8), attn_qkv=np.zeros((24, 8)), attn_proj=np.zeros((8, 8)),
             mlp_fc=np.zeros((16, 8)), mlp_proj=np.zeros((8, 16)))
    cc = draft_model(10, None).cc
    return drafting.DraftModel(cc, [w], capacity, batch=batch, heads=2, dtype=torch.float32, **more)


def i32(x):
    return torch.tensor(x, dtype=torch.int32)


@pytest.mark.parametrize("four", [False, True])
def test_prompts_then_trees(more, four):
    m = model(70, batch=2, cache_bits=4 if four else None)
    got = m.prompt(torch.zeros(9, 8), i32([0, 6, 9]))
    assert got.shape == (9, 8) and m.lens.tolist() == [6, 3]
    assert more == ["prompt", ("fill4", torch.uint8, 12) if four else ("fill", torch.float32, 4)]
    step(m, 5, [2, 1])
    assert more[2:] == (["attention4", "commit4"] if four else ["attention", "commit"]) and m.lens.tolist() == [8, 4]


def test_prompts_that_do_not_fit(more):
    m = model(10, batch=3)
    with pytest.raises(ValueError, match="a prompt of 11 tokens exceeds"):
        m.prompt(torch.zeros(20, 8), i32([0, 4, 15, 20]))
    assert more == [] and m.lens.tolist() == [0, 0, 0]
    m.prompt(torch.zeros(20, 8), i32([0, 4, 14, 20]))
    assert m.lens.tolist() == [4, 10, 6]
    with pytest.raises(ValueError, match="holds rows already"):
        m.prompt(torch.zeros(3, 8), i32([0, 1, 2, 3]))
    # the longest has no room for another node
    with pytest.raises(ValueError, match="10 cached rows and 1 nodes"):
        step(m, 1, [1, 1, 1])


def test_what_does_not_go_together(more):
    with pytest.raises(ValueError, match="cache_bits"):
        model(100, cache_bits=8)
    with pytest.raises(ValueError, match="a 4-bit cache is not cut"):
        model(200, cache_bits=4, budget=100)
    with pytest.raises(ValueError, match="through prefill"):
        model(200, budget=100).prompt(torch.zeros(3, 8), i32([0, 3]))


def test_prefill_into_four_bits(more):
    m = model(100, cache_bits=4)
    m.prefill(torch.zeros(1, 70, 8))
    assert m.lens.tolist() == [70] and more == ["attention4", "commit4"] * 2


@pytest.mark.parametrize("four", [False, True])
def test_prompts_after_the_caches_were_emptied(more, four):
    """Rows that were offered and not accepted, and lengths set back to 0, leave
    room for the next prompts; a single row does not."""
    m = model(20, batch=2, cache_bits=4 if four else None)
    step(m, 3, [0, 0])
    m.prompt(torch.zeros(9, 8), i32([0, 6, 9]))
    assert m.lens.tolist() == [6, 3]
    step(m, 5, [2, 1])
    with pytest.raises(ValueError, match="holds rows already"):
        m.prompt(torch.zeros(9, 8), i32([0, 6, 9]))
    m.lens.zero_()
    m.prompt(torch.zeros(7, 8), i32([0, 0, 7]))
    assert m.lens.tolist() == [0, 7]
    with pytest.raises(ValueError, match="holds rows already"):
        m.prompt(torch.zeros(3, 8), i32([0, 3, 3]))
    step(m, 13, [13, 13])
    assert m.lens.tolist() == [13, 20]


def test_a_4_bit_model_keeps_its_rows_only(more):
    """9/16 of a byte an element, and nothing beside the rows."""
    for (k, v, acc), rest in zip(model(50, batch=2, cache_bits=4).caches, model(50, batch=2).caches):
        assert k.shape == v.shape == (2, 2, 50, 12) and acc is None
        assert rest[0].shape == (2, 2, 50, 4) and rest[2].shape == (2, 2, 50)
