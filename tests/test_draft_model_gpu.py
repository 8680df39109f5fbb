"""Drafted decoding through the framework's models: a tree of drafted tokens
in one encrypted forward, the plain draft model over its cache, and the two
together with the acceptance of the drafts."""

import numpy as np
import pytest

from oracle import plain_block

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import private_genomic_dnagpt_b200 as eng  # noqa: E402
from private_genomic_dnagpt_b200.drafting import DraftModel  # noqa: E402

D, HEADS, MLP, TOKENS = 128, 2, 256, 40


def weights(seed):
    return plain_block.synthetic_weights(seed, d=D, mlp=MLP)


@pytest.fixture(scope="module")
def model():
    cc = eng.GenCryptoContext(eng.CCParams(ring_dim_log=13, limbs=24, dnum=3, seed=51))
    cc.KeyGen()
    cc.EvalMultKeyGen()
    m = eng.EncryptedModel(cc, [weights(52), weights(53)], None, TOKENS, heads=HEADS)
    cc.EvalRotateKeyGen(m.rotation_indices())
    return m


def chain(parents, i):
    return ([] if parents[i] < 0 else chain(parents, parents[i])) + [i]


def plain_tree(x, m, parents, ws):
    """Hidden states of the first m rows and of each node behind its ancestors."""
    rows = [plain_block.model(x[:m], ws, heads=HEADS)[0]]
    for i in range(len(parents)):
        part = np.concatenate([x[:m], x[[m + j for j in chain(parents, i)]]])
        rows.append(plain_block.model(part, ws, heads=HEADS)[0][-1:])
    return np.concatenate(rows)


@pytest.mark.parametrize("first", [31, 20])
def test_encrypted_forward_of_a_tree(model, first):
    parents = [-1, -1, 0, 0, 1, 2, -1, 6, 7]
    ws = [weights(52), weights(53)]
    x = plain_block.synthetic_input(54, TOKENS, d=D)
    hidden, _ = model.forward(x, parents, first if first != 31 else None)
    want = plain_tree(x, first, parents, ws)
    err = plain_block.rel_inf(want, hidden[:first + len(parents)])
    print(f"tree at {first}: rel_inf {err:.3e}")
    assert np.isfinite(hidden).all() and err < 1e-6
    # and causal again afterwards
    causal, _ = model.forward(x)
    assert plain_block.rel_inf(plain_block.model(x, ws, heads=HEADS)[0], causal) < 1e-6


def test_set_drafts_refuses(model):
    b = model.blocks[0]
    for parents, first in (([0], None), ([-1, 1], None), ([-2], None), ([-1] * 65, 0), ([-1], TOKENS), ([-1], -1),
                           ([-1, 0], TOKENS - 1)):
        with pytest.raises(eng.CKKSError):
            b.set_drafts(parents, first)
    b.set_drafts([-1, 0])
    b.set_drafts()


@pytest.mark.parametrize("dtype,tol", [(torch.float32, 1e-4), (torch.bfloat16, 6e-2), (torch.float16, 8e-3)])
def test_draft_model_matches_the_plain_model(model, dtype, tol):
    """Two blocks' hidden states over a prompt and a tree: each block rounds
    its products' operands and results (about 8 roundings deep) to the type,
    a value at most a few times the largest one's half step off."""
    ws = [weights(52), weights(53)]
    x = plain_block.synthetic_input(55, 90, d=D)
    parents = [-1, 0, 0, 1, -1, 4, -1]
    dm = DraftModel(model.cc, ws, capacity=200, heads=HEADS, dtype=dtype)
    t = torch.from_numpy(x).float().cuda()[None]
    p = torch.tensor([parents], dtype=torch.int32, device="cuda")
    got = [dm.prefill(t[:, :83]), dm.forward(t[:, 83:], p)]
    assert int(dm.lens[0]) == 83
    want = plain_tree(x, 83, parents, ws)
    assert plain_block.rel_inf(want, torch.cat(got, 1)[0].double().cpu().numpy()) < tol
    # nodes 0 and 2 accepted: the next token follows them
    dm.accept(torch.tensor([[0, 2] + [-1] * 5], dtype=torch.int32, device="cuda"),
              torch.tensor([2], dtype=torch.int32, device="cuda"))
    one = torch.tensor([[-1]], dtype=torch.int32, device="cuda")
    nxt = dm.forward(t[:, 5:6], one)[0].double().cpu().numpy()
    seq = np.concatenate([x[:83], x[[83, 85]], x[5:6]])
    assert plain_block.rel_inf(plain_block.model(seq, ws, heads=HEADS)[0][-1:], nxt) < tol
    model.cc.Synchronize()


def test_draft_model_keeps_to_its_budget(model):
    """The cache is cut when a tree would not fit, and holds the latest rows
    and those that the definitions give the most weight."""
    ws = [weights(56)]
    x = torch.from_numpy(plain_block.synthetic_input(57, 200, d=D)).float().cuda()[None]
    small = DraftModel(model.cc, ws, capacity=164, heads=HEADS, dtype=torch.float32, budget=100, recent=20)
    large = DraftModel(model.cc, ws, capacity=264, heads=HEADS, dtype=torch.float32, budget=200, recent=20)
    small.prefill(x[:, :128])
    large.prefill(x[:, :128])
    assert int(small.lens[0]) == 128
    small.prefill(x[:, 128:140])
    assert int(small.lens[0]) == 140 and small._most == 140
    small.forward(x[:, 140:170], torch.arange(-1, 29, dtype=torch.int32, device="cuda")[None])  # 140 + 30 > 164
    assert int(small.lens[0]) == 100
    large.prefill(x[:, 128:140])
    k, v, acc = large.caches[0]
    for h in range(HEADS):
        w = acc[0, h, :120]
        heavy = torch.sort(w, descending=True, stable=True).indices[:80].sort().values
        rows = torch.cat([heavy, torch.arange(120, 140, device="cuda")])
        assert torch.equal(small.caches[0][0][0, h, :100], k[0, h, rows])
        assert torch.equal(small.caches[0][1][0, h, :100], v[0, h, rows])
    full = DraftModel(model.cc, ws, capacity=70, heads=HEADS, dtype=torch.float32)
    full.prefill(x[:, :64])
    with pytest.raises(ValueError, match="exceed the capacity"):
        full.forward(x[:, :7], torch.full((1, 7), -1, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError, match="do not fit"):
        DraftModel(model.cc, ws, capacity=100, heads=HEADS, budget=50)
    model.cc.Synchronize()


def test_draft_model_of_a_batch(model):
    """Two sequences side by side, with trees of different sizes and other
    accepted nodes, as two models of one."""
    ws = [weights(60), weights(61)]
    x = torch.from_numpy(np.stack([plain_block.synthetic_input(s, 100, d=D) for s in (62, 63)])).float().cuda()
    both = DraftModel(model.cc, ws, capacity=164, batch=2, heads=HEADS, dtype=torch.float32, budget=100, recent=10)
    ones = [DraftModel(model.cc, ws, capacity=164, heads=HEADS, dtype=torch.float32, budget=100, recent=10)
            for _ in range(2)]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    parents, path, count = [[-1, 0, 0, 1], [-1, -1, -2, 2]], [[0, 1, 3, -1], [1, -1, -1, -1]], [3, 1]
    both.prefill(x[:, :60])
    for m, s in zip(ones, x):
        m.prefill(s[None, :60])
    for step in range(4):
        rows = x[:, 60 + 4 * step:64 + 4 * step]
        got = both.forward(rows, i32(parents))
        both.accept(i32(path), i32(count))
        for b, m in enumerate(ones):
            want = m.forward(rows[b:b + 1], i32(parents[b:b + 1]))
            real = 4 if b == 0 else 2
            assert (got[b, :real] - want[0, :real]).abs().max() <= 1e-5 * want.abs().max()
            m.accept(i32(path[b:b + 1]), i32(count[b:b + 1]))
    assert both.lens.tolist() == [72, 64] == [int(m.lens[0]) for m in ones]
    for (k, v, acc), pairs in zip(both.caches, zip(ones[0].caches, ones[1].caches)):
        for b, (k1, v1, a1) in enumerate(pairs):
            n = int(both.lens[b])
            for t, t1 in ((k, k1), (v, v1), (acc, a1)):
                assert (t[b, :, :n] - t1[0, :, :n]).abs().max() <= 1e-4 * t1[0, :, :n].abs().max()
    model.cc.Synchronize()


def test_drafts_confirmed_by_the_encrypted_model(model):
    """The whole round: the draft model proposes a tree of greedy tokens, the
    encrypted model evaluates it in one forward, the accepted nodes enter the
    cache, and the tokens are those that the plain target model gives."""
    ws, V = [weights(52), weights(53)], 50
    rng = np.random.default_rng(58)
    table, readout = plain_block.synthetic_input(59, V, d=D), 3.0 * rng.standard_normal((V, D))
    context = list(rng.integers(0, V, 12))
    # the target's weights, a little off
    dm = DraftModel(model.cc, [{k: v + 2e-4 * rng.standard_normal(v.shape) for k, v in w.items()} for w in ws],
                    capacity=200, heads=HEADS, dtype=torch.float32)
    emb = torch.from_numpy(table).float().cuda()
    out = torch.from_numpy(readout).cuda()
    i32 = lambda v: torch.tensor([v], dtype=torch.int32, device="cuda")  # noqa: E731
    hidden = dm.prefill(emb[context][None])[0, -1]
    took = []
    for _ in range(2):
        # a chain of three most likely tokens, each with its runner-up as a sibling
        tokens, parents, probs, last, path = [], [], [], -1, []
        h = hidden
        for _ in range(3):
            p = torch.softmax(h.double() @ out.T, -1)
            best = p.topk(2).indices.tolist()
            tokens += best
            parents += [last, last]
            last = len(tokens) - 2
            path.append(last)
            nodes = dm.forward(emb[tokens][None], i32(parents))[0]
            h = nodes[last]
        n = len(tokens)
        # the drafts are certain choices: q is 1 for the first child and, where it is refused, for the second
        q = np.zeros((n + 1, V))
        for i, par in enumerate(parents):
            if i % 2 == 0:
                q[par + 1, tokens[i]] = 1.0
        uniforms = rng.random(n + 1)
        got, token = model.verify_drafts(table[context], table[tokens], tokens, parents, q, uniforms, readout)
        want_hidden = plain_tree(np.concatenate([table[context], table[tokens]]), len(context), parents, ws)
        logits = want_hidden[len(context) - 1:] @ readout.T
        target = np.exp(logits - logits.max(-1, keepdims=True))
        target /= target.sum(-1, keepdims=True)
        import draft_reference as ref
        wp, wc, wt = ref.verify(target[None], q[None], np.array([tokens]), np.array([parents]), uniforms[None])
        assert got == wp[0, :wc[0]].tolist() and token == wt[0]
        dm.accept(i32(got + [-1] * (n - len(got))), torch.tensor([len(got)], dtype=torch.int32, device="cuda"))
        context += [tokens[i] for i in got]
        assert int(dm.lens[0]) == len(context)
        hidden = dm.forward(emb[[token]][None], i32([-1]))[0, -1]
        dm.accept(i32([0]), torch.tensor([1], dtype=torch.int32, device="cuda"))
        context.append(token)
        took.append(len(got) + 1)
        plain = plain_block.model(table[context], ws, heads=HEADS)[0][-1]
        assert plain_block.rel_inf(plain, hidden.double().cpu().numpy()) < 0.05
    print("tokens per encrypted forward:", took)
    model.cc.Synchronize()
