"""DraftModel over packed prompts and 4-bit caches: a run of prompt, tree and
commit against the blocks in float64, on rows that the cache has rounded."""

import numpy as np
import pytest

import prompt_reference as ref
from oracle import plain_block

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import private_genomic_dnagpt_b200 as eng  # noqa: E402
from private_genomic_dnagpt_b200.drafting import DraftModel  # noqa: E402

from test_draft_gpu import f64, i32, tree  # noqa: E402

D, HEADS, MLP = 128, 2, 256


@pytest.fixture(scope="module")
def cc():
    return eng.GenCryptoContext(eng.CCParams(ring_dim_log=10, limbs=3, dnum=1, seed=3))


def weights(seed):
    w = plain_block.synthetic_weights(seed, d=D, mlp=MLP)
    return {k: np.float32(v) for k, v in w.items()}


def norm(x, w):
    x = x - x.mean(-1, keepdims=True)
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-5) * w


def gelu(x):
    return 0.5 * x * (1 + np.tanh(np.sqrt(2 / np.pi) * (x + 0.044715 * x ** 3)))


class Plain:
    """One sequence in float64: each block's cached keys and values, which are
    rounded to 4 bits as they enter where `four` is set."""

    def __init__(self, ws, four):
        self.ws, self.four = ws, four
        self.k, self.v = ([np.zeros((0, HEADS, D // HEADS)) for _ in ws] for _ in range(2))

    def forward(self, x, parents):
        """parents of a prompt: a chain."""
        self.new = []
        see = [[i] for i in range(len(parents))]
        for i, p in enumerate(parents):
            see[i] += see[p] if p >= 0 else []
        for w, k0, v0 in zip(self.ws, self.k, self.v):
            q, k, v = (norm(x, w["ln1"]) @ w["attn_qkv"].T).reshape(len(x), 3, HEADS, -1).swapaxes(0, 1)
            out = np.zeros_like(q)
            for i in range(len(x)):
                kk, vv = np.concatenate([k0, k[see[i]]]), np.concatenate([v0, v[see[i]]])
                s = np.einsum("hd,khd->hk", q[i], kk) / np.sqrt(D // HEADS)
                p = np.exp(s - s.max(1, keepdims=True))
                out[i] = np.einsum("hk,khd->hd", p / p.sum(1, keepdims=True), vv)
            x = x + out.reshape(len(x), D) @ w["attn_proj"].T
            x = x + gelu(norm(x, w["ln2"]) @ w["mlp_fc"].T) @ w["mlp_proj"].T
            self.new.append((k, v))
        return x

    def accept(self, path):
        held = (lambda y: ref.unpack(ref.pack(y), D // HEADS)) if self.four else (lambda y: y)
        self.k = [np.concatenate([c, held(n[0][path])]) for c, n in zip(self.k, self.new)]
        self.v = [np.concatenate([c, held(n[1][path])]) for c, n in zip(self.v, self.new)]


@pytest.mark.parametrize("four", [False, True])
def test_prompts_trees_and_commits(cc, four):
    """Packed prompts of three lengths, two rounds of trees behind them."""
    ws = [weights(70), weights(71)]
    lengths, n = [37, 1, 150], 7
    starts = [0, 37, 38, 188]
    x = np.float32(plain_block.synthetic_input(72, 250, d=D))
    m = DraftModel(cc, ws, capacity=200, batch=3, heads=HEADS, dtype=torch.float32, cache_bits=4 if four else None)
    plain = [Plain([{k: v.astype(np.float64) for k, v in w.items()} for w in ws], four) for _ in lengths]
    cuda = lambda y: torch.from_numpy(np.ascontiguousarray(y)).cuda()  # noqa: E731
    got = f64(m.prompt(cuda(x[:188]), i32(starts)))
    for p, a, e in zip(plain, starts, starts[1:]):
        want = p.forward(x[a:e].astype(np.float64), list(range(-1, e - a - 1)))
        p.accept(list(range(e - a)))
        assert plain_block.rel_inf(want, got[a:e]) < 1e-4
    # a code may differ where float32 keys lie next to a border; the rows agree but for such
    if four:
        for b, p in enumerate(plain):
            rows = m.caches[0][0][b, :, :len(p.k[0])].cpu().numpy()
            values = ref.unpack(rows, D // HEADS)
            assert (values == p.k[0].swapaxes(0, 1)).mean() > 0.999
            # from here on both have the same rows
            for i, (kc, vc, _) in enumerate(m.caches):
                p.k[i], p.v[i] = (ref.unpack(c[b, :, :lengths[b]].cpu().numpy(), D // HEADS).swapaxes(0, 1) for c in (kc, vc))
    parents = tree(n, 2)
    for step in range(2):
        nodes = x[190 + n * step:190 + n * (step + 1)]
        got = f64(m.forward(cuda(np.stack([nodes] * 3)), i32([parents] * 3)))
        path = [0, 2, 5]
        for b, p in enumerate(plain):
            want = p.forward(nodes.astype(np.float64), parents)
            assert plain_block.rel_inf(want, got[b]) < (5e-3 if four and step else 1e-4)
            p.accept(path[:b + 1])
        m.accept(i32([path + [-1] * (n - 3)] * 3), i32([1, 2, 3]))
    assert m.lens.tolist() == [37 + 2, 1 + 4, 150 + 6] == [len(p.k[0]) for p in plain]
    cc.Synchronize()


@pytest.mark.parametrize("dtype,most", [(torch.float32, 2e-5), (torch.bfloat16, 0.05), (torch.float16, 0.01)])
def test_prompt_and_prefill_agree(cc, dtype, most):
    """The same prompt through ``prompt`` and through ``prefill``'s trees."""
    ws = [weights(73), weights(74)]
    x = torch.from_numpy(np.float32(plain_block.synthetic_input(75, 200, d=D))).cuda()
    a, b = (DraftModel(cc, ws, capacity=264, heads=HEADS, dtype=dtype) for _ in range(2))
    got, want = a.prompt(x, i32([0, 200])), b.prefill(x[None])[0]
    assert plain_block.rel_inf(f64(want), f64(got)) < most
    assert a.lens.tolist() == b.lens.tolist() == [200]
    for (k, v, _), (k2, v2, _) in zip(a.caches, b.caches):
        for c, c2 in ((k, k2), (v, v2)):
            assert (c[:, :, :200].float() - c2[:, :, :200].float()).abs().max() <= most * c2.float().abs().max()
            assert not c[:, :, 200:].any()
    nodes = x[None, :5]
    chain = i32([[-1, 0, 1, 2, 3]])
    assert plain_block.rel_inf(f64(b.forward(nodes, chain)), f64(a.forward(nodes, chain))) < most
    cc.Synchronize()


@pytest.mark.parametrize("dtype,most", [(torch.bfloat16, 0.05), (torch.float16, 0.01)])
def test_four_bits_in_the_16_bit_types(cc, dtype, most):
    """The default type: prompt, trees and commits over a 4-bit cache against the
    same model over a plain cache that is given the values of the other's."""
    ws = [weights(76), weights(77)]
    x = torch.from_numpy(np.float32(plain_block.synthetic_input(78, 300, d=D))).cuda()
    starts, n = [0, 150, 151, 260], 7
    a = DraftModel(cc, ws, capacity=200, batch=3, heads=HEADS, dtype=dtype, cache_bits=4)
    b = DraftModel(cc, ws, capacity=200, batch=3, heads=HEADS, dtype=dtype)
    got, want = a.prompt(x[:260], i32(starts)), b.prompt(x[:260], i32(starts))
    assert torch.equal(got, want)  # attention within the prompts reads no cache

    def give():
        for (k4, v4, _), (k, v, _) in zip(a.caches, b.caches):
            k.copy_(cc.draft_read4(k4, a.lens, D // HEADS, dtype))
            v.copy_(cc.draft_read4(v4, a.lens, D // HEADS, dtype))

    for step in range(2):
        give()
        nodes = x[260 + n * step:260 + n * (step + 1)].repeat(3, 1, 1)
        got, want = (m.forward(nodes, i32([tree(n, 2)] * 3)) for m in (a, b))
        assert plain_block.rel_inf(f64(want), f64(got)) < most
        for m in (a, b):
            m.accept(i32([[0, 2, 5, -1, -1, -1, -1]] * 3), i32([3, 0, 1]))
        assert a.lens.tolist() == b.lens.tolist() == [150 + 3 * (step + 1), 1, 109 + step + 1]
    cc.Synchronize()


@pytest.mark.parametrize("four", [False, True])
def test_a_model_serves_batch_after_batch(cc, four):
    """Emptied caches give the results of new ones."""
    ws = [weights(79), weights(80)]
    x = torch.from_numpy(np.float32(plain_block.synthetic_input(81, 200, d=D))).cuda()
    used = DraftModel(cc, ws, capacity=128, batch=2, heads=HEADS, cache_bits=4 if four else None)
    chain = i32([[-1, 0, 1]] * 2)
    for lengths in ([90, 20], [3, 120], [0, 70]):
        new = DraftModel(cc, ws, capacity=128, batch=2, heads=HEADS, cache_bits=4 if four else None)
        starts, nodes = i32([0, lengths[0], sum(lengths)]), x[150:153].repeat(2, 1, 1)
        used.lens.zero_()
        got, want = (m.prompt(x[:sum(lengths)], starts) for m in (used, new))
        assert torch.equal(got, want)
        got, want = (m.forward(nodes, chain) for m in (used, new))
        assert torch.equal(got, want)
        for m in (used, new):
            m.accept(chain + 1, i32([3, 1]))
        assert used.lens.tolist() == new.lens.tolist() == [lengths[0] + 3, lengths[1] + 1]
    cc.Synchronize()
