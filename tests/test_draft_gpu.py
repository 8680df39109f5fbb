"""The drafted-decoding operators on the GPU against their definitions in
float64 (tests/draft_reference.py).

Bounds: u is half a step of the tensors' type (2^-8 bfloat16, 2^-11 float16,
2^-24 float32).  A row's result is a sum of p_k v_k: the weights may be rounded
to the type (u), the result is (u), the scores carry D + 8 roundings of
2^-24 on sum |q k| scale, and a sum over N keys N + 8 more, each at most
doubled by the division through a sum with the same error.  So
|out - exact| <= (2 u + 2^-23 ((D + 8) S + N + 8)) sum p |v| with
S = sum |q k| scale, and lse is off by half of the second part plus 2^-22 of
itself."""

import ctypes

import numpy as np
import pytest

import draft_reference as ref

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import private_genomic_dnagpt_b200 as eng  # noqa: E402

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture(scope="module")
def cc():
    return eng.GenCryptoContext(eng.CCParams(ring_dim_log=10, limbs=3, dnum=1, seed=3))


def f64(t):
    return t.detach().to(torch.float64).cpu().numpy()


def tree(n, branch, pad=0):
    return [i // branch - 1 if i < n - pad else -2 for i in range(n)]


def i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def inputs(dtype, B, n, Hq, Hk, D, cap, lens, parents, seed=0, spread=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *s: (spread * torch.randn(*s, generator=g, device="cuda")).to(dtype)  # noqa: E731
    return dict(q=normal(B, n, Hq, D), k_cache=normal(B, Hk, cap, D), v_cache=normal(B, Hk, cap, D), lens=i32(lens),
                k_new=normal(B, n, Hk, D), v_new=normal(B, n, Hk, D), parents=i32(parents))


def check_attention(x, out, lse, scale=None):
    q = f64(x["q"])
    D = q.shape[3]
    scale = D ** -0.5 if scale is None else scale
    want, wlse, mag, big, keys = ref.attention(q, f64(x["k_cache"]), f64(x["v_cache"]), x["lens"].cpu().numpy(),
                                               f64(x["k_new"]), f64(x["v_new"]), x["parents"].cpu().numpy(), scale)
    got, glse = f64(out), f64(lse)
    noise = 2.0 ** -23 * ((D + 8) * big + keys + 8)
    room = (2 * HALF[x["q"].dtype] + noise)[..., None] * mag + 1e-30
    assert np.array_equal(np.isfinite(want), np.isfinite(got))
    fine = np.isfinite(want)
    worst = (np.abs(got - want)[fine] / room[fine]).max() if fine.any() else 0.0
    assert worst <= 1.0, f"out: {worst:.3g} times the bound"
    seen = keys > 0
    assert np.array_equal(glse == -np.inf, ~seen)
    off = np.abs(glse[seen] - wlse[seen])
    assert (off <= (0.5 * noise + 2.0 ** -22 * (1 + np.abs(wlse)))[seen]).all()
    assert not got[~seen].any()


SHAPES = [
    # B, n, Hq, Hk, D, cap, lens, branch, pad
    (1, 1, 12, 12, 64, 128, [103], 1, 0),
    (1, 1, 1, 1, 64, 1, [0], 1, 0),            # no cached key: the node sees itself
    (1, 1, 2, 1, 64, 1, [1], 1, 0),
    (3, 5, 4, 2, 64, 200, [200, 0, 77], 1, 0),
    (2, 21, 12, 12, 64, 700, [640, 511], 2, 2),
    (2, 64, 4, 4, 64, 333, [333, 128], 2, 0),  # the largest tree
    (2, 64, 4, 1, 128, 300, [257, 300], 3, 1),  # 256 rows on one key/value head
    (1, 33, 8, 2, 128, 1500, [1493], 4, 0),
    (2, 7, 6, 3, 32, 130, [129, 64], 2, 0),
    (1, 9, 4, 2, 80, 190, [190], 3, 0),
    (2, 4, 2, 2, 96, 300, [255, 256], 1, 0),
    (1, 3, 2, 1, 256, 140, [131], 1, 0),
    (1, 6, 3, 3, 192, 100, [99], 2, 0),
    (2, 3, 2, 2, 1, 50, [50, 3], 1, 0),
    (1, 5, 2, 1, 5, 70, [66], 2, 0),
    (1, 2, 5, 5, 33, 90, [65], 1, 0),
    (1, 2, 2, 2, 40, 70, [64], 1, 0),
    (1, 64, 1, 1, 64, 4, [3], 1, 0),           # a chain of 64
    (1, 64, 2, 2, 64, 0, [0], 2, 0),           # a cache without rows
    (1, 2, 1, 1, 64, 70000, [200], 1, 0),      # far more capacity than keys
    (5, 1, 1, 1, 64, 50000, [0] * 5, 1, 0),
    (1, 3, 130, 1, 64, 150, [140], 1, 0),      # more heads on a key than a tile has rows
    (1, 2, 128, 1, 128, 150, [129], 1, 0),
    (2, 64, 6, 2, 64, 260, [257, 3], 3, 1),    # tiles of 126 rows
    (1, 5, 96, 2, 32, 140, [133], 2, 0),
    (1, 12, 8, 1, 80, 900, [897], 2, 0),       # 96 rows
    (2, 40, 8, 2, 256, 900, [897, 300], 2, 1),
    (3, 64, 4, 1, 160, 700, [700, 0, 129], 3, 2),
    (2, 17, 3, 3, 136, 1000, [999, 640], 2, 0),
    (1, 33, 2, 1, 192, 2000, [1999], 1, 0),
    (70, 9, 2, 2, 248, 260, [(53 * b) % 261 for b in range(70)], 2, 0),
    (3, 3, 2, 1, 128, 40000, [129, 0, 300], 1, 1),
    (40, 2, 2, 1, 64, 300, [(37 * b) % 301 for b in range(40)], 1, 0),  # many short sequences
    (70, 33, 2, 2, 64, 140, [(53 * b) % 141 for b in range(70)], 2, 0),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_attention(cc, dtype, shape):
    B, n, Hq, Hk, D, cap, lens, branch, pad = shape
    x = inputs(dtype, B, n, Hq, Hk, D, cap, lens, [tree(n, branch, pad if b == B - 1 else 0) for b in range(B)])
    check_attention(x, *cc.draft_attention(**x))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(2, 13, 8, 2, 128, 9000, [8999, 4097], 3), (1, 1, 4, 4, 64, 20000, [19999], 1),
                                   (1, 40, 4, 1, 64, 5000, [4999], 2),
                                   (2, 21, 4, 1, 256, 9000, [8999, 4097], 3)])
def test_attention_over_long_caches(cc, dtype, shape):
    B, n, Hq, Hk, D, cap, lens, branch = shape
    x = inputs(dtype, B, n, Hq, Hk, D, cap, lens, [tree(n, branch)] * B, seed=1)
    check_attention(x, *cc.draft_attention(**x))


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_sharp_rows(cc, dtype):
    """Scores far apart: the running maximum moves by hundreds."""
    x = inputs(dtype, 2, 6, 4, 2, 64, 600, [600, 321], [tree(6, 2)] * 2, seed=2, spread=6.0)
    check_attention(x, *cc.draft_attention(**x))
    check_attention(x, *cc.draft_attention(**x, scale=0.5), scale=0.5)
    check_attention(x, *cc.draft_attention(**x, scale=-0.01), scale=-0.01)
    check_attention(x, *cc.draft_attention(**x, scale=0.0), scale=0.0)
    x = inputs(dtype, 2, 6, 4, 2, 200, 600, [600, 321], [tree(6, 2)] * 2, seed=2, spread=6.0)
    check_attention(x, *cc.draft_attention(**x))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("D", [64, 128, 40, 256])
def test_attention_ignores_what_is_masked(cc, dtype, bad, D):
    """Rows behind the length and padding nodes hold NaN and infinities."""
    lens = [130, 0, 257]
    x = inputs(dtype, 3, 10, 4, 2, D, 300, lens, [tree(10, 2, 3)] * 3, seed=4)
    clean = cc.draft_attention(**x)
    for b, m in enumerate(lens):
        x["k_cache"][b, :, m:] = bad
        x["v_cache"][b, :, m:] = bad
    x["k_new"][:, 7:] = bad
    x["v_new"][:, 7:] = bad
    x["q"][:, 7:] = bad
    got = cc.draft_attention(**x)
    assert torch.equal(clean[0], got[0]) and torch.equal(clean[1], got[1])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 128, 40, 256])
@pytest.mark.parametrize("G", [1, 4])
def test_attention_keeps_siblings_apart(cc, dtype, D, G):
    """A node whose key and value are NaN or infinite spoils its own row and
    its children's, not its siblings'."""
    parents = [-1, -1, 0, 0, 1, 1, 4]
    x = inputs(dtype, 2, 7, 2 * G, 2, D, 200, [190, 0], [parents] * 2, seed=5)
    clean = f64(cc.draft_attention(**x)[0])
    x["k_new"][:, 1] = float("nan")
    x["v_new"][:, 1] = float("nan")
    x["v_new"][:, 3] = float("inf")
    got, lse = (f64(t) for t in cc.draft_attention(**x))
    for i in (0, 2):
        assert np.array_equal(got[:, i], clean[:, i])
    for i in (1, 4, 5, 6):
        assert np.isnan(got[:, i]).all() and np.isnan(lse[:, i]).all()
    assert (got[:, 3] == np.inf).all() and np.isfinite(lse[:, 3]).all()


def test_attention_odd_parents(cc):
    """A parent that is not an earlier node makes padding of the node and of
    what hangs below it."""
    parents = [[-1, 1, 0, 3, 2, 7, -5, 2 ** 31 - 1], [-2, 0, -1, 2, 2, 1, 5, -2 ** 31]]
    x = inputs(torch.bfloat16, 2, 8, 2, 2, 64, 100, [100, 70], parents, seed=6)
    out, lse = cc.draft_attention(**x)
    check_attention(x, out, lse)
    assert torch.isinf(lse[0, [1, 3, 5, 6, 7]]).all() and torch.isinf(lse[1, [0, 1, 5, 6, 7]]).all()


def test_attention_lengths_are_clamped(cc):
    x = inputs(torch.float16, 3, 2, 2, 2, 64, 96, [500, -3, 96], [tree(2, 1)] * 3, seed=7)
    check_attention(x, *cc.draft_attention(**x))


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_strides_and_alignment(cc, dtype):
    x = inputs(dtype, 2, 6, 4, 2, 64, 210, [200, 111], [tree(6, 2)] * 2, seed=8)
    want = cc.draft_attention(**x)
    y = dict(x)
    y["k_cache"] = x["k_cache"].transpose(1, 2).contiguous().transpose(1, 2)      # rows of the heads interleaved
    wide = torch.zeros(2, 2, 210, 72, dtype=dtype, device="cuda")
    wide[..., :64] = x["v_cache"]
    y["v_cache"] = wide[..., :64]
    y["q"] = x["q"].transpose(1, 2).contiguous().transpose(1, 2)
    y["k_new"] = x["k_new"].transpose(1, 2).contiguous().transpose(1, 2)
    got = cc.draft_attention(**y)
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
    for name in ("q", "k_cache", "v_cache", "k_new", "v_new"):  # one element off every wide boundary
        flat = torch.zeros(x[name].numel() + 1, dtype=dtype, device="cuda")
        flat[1:] = x[name].reshape(-1)
        z = dict(x) | {name: flat[1:].view(x[name].shape)}
        check_attention(z, *cc.draft_attention(**z))
    one = dict(x) | {"k_cache": x["k_cache"][:1].expand(2, 2, 210, 64)}  # one cache for both sequences
    check_attention(one, *cc.draft_attention(**one))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_offsets_past_32_bits(cc, dtype):
    """Rows 2^25 elements apart: the last ones lie past 2^31 elements."""
    step, cap = 1 << 25, 70
    store = torch.empty(step * cap, dtype=dtype, device="cuda")
    x = inputs(dtype, 1, 3, 2, 2, 64, cap, [cap], [tree(3, 1)], seed=9)
    for name, at in (("k_cache", 0), ("v_cache", 4096)):
        view = torch.as_strided(store, (1, 2, cap, 64), (128, 64, step, 1), at)
        view.copy_(x[name])
        x[name] = view
    check_attention(x, *cc.draft_attention(**x))


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_repeats_exactly(cc, dtype):
    x = inputs(dtype, 2, 21, 8, 2, 128, 5000, [5000, 3333], [tree(21, 2)] * 2, seed=10)
    a, b = cc.draft_attention(**x), cc.draft_attention(**x)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 64), (torch.float16, 128), (torch.float32, 64), (torch.float32, 33)])
def test_attention_on_other_streams_and_in_graphs(cc, dtype, D):
    """Two captured calls replayed side by side, and one on another stream."""
    xs = [inputs(dtype, 1, 5, 4, 4, D, 6000, [5999 - s], [tree(5, 1)], seed=11 + s) for s in range(2)]
    want = [cc.draft_attention(**x) for x in xs]
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = cc.draft_attention(**xs[0])
    s.synchronize()
    assert torch.equal(got[0], want[0][0])
    graphs, outs = [], []
    for x in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(cc.draft_attention(**x))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in xs]
    for o in outs:
        o[0].zero_()
    torch.cuda.synchronize()
    for _ in range(20):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert torch.equal(o[0], w[0]) and torch.equal(o[1], w[1])


def test_attention_empty_batch(cc):
    x = inputs(torch.bfloat16, 0, 3, 2, 2, 64, 10, np.zeros(0), np.zeros((0, 3)))
    out, lse = cc.draft_attention(**x)
    assert out.shape == (0, 3, 2, 64) and lse.shape == (0, 3, 2)


# ---- verify ---------------------------------------------------------------------

def verify_inputs(B, n, V, branch, tt, td, seed, noise=0.7, pad=0):
    rng = np.random.default_rng(seed)
    logits = 2.5 * rng.standard_normal((B, n + 1, V))
    other = logits + noise * rng.standard_normal((B, n + 1, V))
    soft = lambda x: np.exp(x - x.max(-1, keepdims=True)) / np.exp(x - x.max(-1, keepdims=True)).sum(-1, keepdims=True)  # noqa: E731,E501
    target = torch.tensor(soft(logits), dtype=tt, device="cuda")
    draft = torch.tensor(soft(other), dtype=td, device="cuda")
    parents = np.array([tree(n, branch, pad)] * B)
    d = f64(draft)
    tokens = np.zeros((B, n), int)
    for b in range(B):
        for i in range(n):
            p = d[b, max(0, parents[b, i] + 1)]
            tokens[b, i] = rng.choice(V, p=p / p.sum())
    return dict(target=target, draft=draft, tokens=i32(tokens), parents=i32(parents),
                uniforms=torch.tensor(rng.random((B, n + 1)), device="cuda"))


def check_verify(cc, x):
    path, count, token = (t.cpu().numpy() for t in cc.draft_verify(**x))
    want = ref.verify(f64(x["target"]), f64(x["draft"]), x["tokens"].cpu().numpy(), x["parents"].cpu().numpy(),
                      f64(x["uniforms"]))
    assert np.array_equal(path, want[0]) and np.array_equal(count, want[1]) and np.array_equal(token, want[2])
    return path, count, token


@pytest.mark.parametrize("tt,td", [(torch.float32, torch.float32), (torch.float64, torch.float64),
                                   (torch.float64, torch.float32), (torch.float32, torch.float64)])
@pytest.mark.parametrize("B,n,V,branch,pad", [(1, 5, 4103, 1, 0), (9, 31, 1000, 2, 2), (7, 12, 33, 4, 0),
                                              (5, 1, 1, 1, 0), (6, 64, 7, 8, 1), (4, 8, 1024, 8, 0),
                                              (2, 3, 40001, 1, 0), (3, 20, 32, 64, 0), (3, 6, 1025, 2, 0),
                                              (2, 5, 128256, 2, 0), (1, 4, 300007, 1, 0), (40, 7, 8200, 2, 0)])
def test_verify(cc, tt, td, B, n, V, branch, pad):
    counts = []
    for seed in range(4):
        counts += list(check_verify(cc, verify_inputs(B, n, V, branch, tt, td, 10 * seed + 1, pad=pad))[1])
    assert max(counts) > 0


def test_verify_all_accepted_and_all_refused(cc):
    x = verify_inputs(4, 6, 500, 1, torch.float64, torch.float64, 3)
    same = dict(x) | {"draft": x["target"].clone(), "tokens": x["tokens"]}
    same["uniforms"][:, :6] = 0.999999
    assert (check_verify(cc, same)[1] == 6).all()  # p = q: always accepted
    none = dict(x)
    target = x["target"].clone()
    for i in range(6):  # the target gives the first draft nothing
        target[torch.arange(4), i, x["tokens"][:, i].long()] = 0.0
    none["target"] = target
    assert (check_verify(cc, none)[1] == 0).all()


def test_verify_siblings_share_one_row(cc):
    """Up to 64 children of the root, the same token among them twice."""
    x = verify_inputs(8, 64, 300, 64, torch.float64, torch.float32, 5, noise=2.5)
    x["tokens"][:, 1] = x["tokens"][:, 0]
    check_verify(cc, x)
    x["uniforms"][:, :63] = 0.9999
    check_verify(cc, x)


def test_verify_greedy_rows(cc):
    """One-hot targets: exactly the drafts that are the target's choice."""
    x = verify_inputs(6, 4, 97, 1, torch.float32, torch.float32, 6)
    best = x["target"].argmax(-1)
    x["target"] = torch.nn.functional.one_hot(best, 97).float()
    x["tokens"][:3] = best[:3, :4].int()
    x["tokens"][0, 2] = (best[0, 2] + 1) % 97
    _, count, token = check_verify(cc, x)
    assert list(count[:3]) == [2, 4, 4] and token[0] == int(best[0, 2])


def test_verify_edges(cc):
    x = verify_inputs(6, 5, 130, 2, torch.float64, torch.float64, 7)
    x["tokens"][0, :2] = torch.tensor([130, -1], dtype=torch.int32)   # outside the vocabulary
    x["tokens"][1, 0] = 2 ** 31 - 1
    x["uniforms"][2] = 0.0
    x["uniforms"][3] = 1.0 - 2.0 ** -53
    x["target"][4, 0] = 0.0                                            # a row without weight
    x["target"][5, :, 3] = float("nan")
    x["draft"][5, :, 4] = -1.0
    check_verify(cc, x)


def test_verify_strides(cc):
    x = verify_inputs(3, 4, 77, 2, torch.float32, torch.float64, 8)
    want = cc.draft_verify(**x)
    y = dict(x)
    wide = torch.zeros(3, 5, 90, device="cuda")
    wide[..., 1:78] = x["target"]
    y["target"] = wide[..., 1:78]
    y["draft"] = x["draft"].transpose(0, 1).contiguous().transpose(0, 1)
    assert all(torch.equal(a, b) for a, b in zip(want, cc.draft_verify(**y)))


def test_verify_distribution(cc):
    """The first token kept is distributed as the target's row: each of 5
    tokens within five standard deviations over 40000 trials."""
    B, V = 40000, 5
    rng = np.random.default_rng(9)
    p, q = np.array([0.05, 0.3, 0.4, 0.05, 0.2]), np.array([0.4, 0.1, 0.3, 0.15, 0.05])
    tokens = rng.choice(V, size=(B, 3), p=q)
    x = dict(target=torch.tensor(p, device="cuda").expand(B, 4, V), draft=torch.tensor(q, device="cuda").expand(B, 4, V),
             tokens=i32(tokens), parents=i32([[-1, -1, -1]] * B), uniforms=torch.tensor(rng.random((B, 4)), device="cuda"))
    path, count, token = (t.cpu().numpy() for t in cc.draft_verify(**x))
    first = np.where(count > 0, tokens[np.arange(B), np.maximum(path[:, 0], 0)], token)
    share = np.bincount(first, minlength=V) / B
    assert (np.abs(share - p) < 5 * np.sqrt(p * (1 - p) / B)).all()


# ---- commit, accumulate, evict ------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 40, 33, 1])
def test_commit(cc, dtype, D):
    B, n, Hk, cap = 5, 9, 3, 60
    lens, count = [0, 10, 51, 57, 60], [9, 3, 9, 3, 0]
    x = inputs(dtype, B, n, Hk, Hk, D, cap, lens, [tree(n, 2)] * B, seed=12)
    path = np.array([[8, 8, 0, 1, 2, 3, 4, 5, 6], [0, 2, 6] + [-1] * 6, list(range(9)), [1, 3, 7] + [-1] * 6, [-1] * 9])
    want = {k: x[k].clone() for k in ("k_cache", "v_cache")}
    for b in range(B):
        for j in range(count[b]):
            for c, f in (("k_cache", "k_new"), ("v_cache", "v_new")):
                want[c][b, :, lens[b] + j] = x[f][b, path[b, j]]
    new = cc.draft_commit(x["k_cache"], x["v_cache"], x["lens"], x["k_new"], x["v_new"], i32(path), i32(count))
    assert new.tolist() == [a + b for a, b in zip(lens, count)]
    assert torch.equal(x["k_cache"], want["k_cache"]) and torch.equal(x["v_cache"], want["v_cache"])
    cc.Synchronize()


def test_commit_leaves_what_does_not_fit(cc):
    B, n, Hk, D, cap = 7, 4, 2, 64, 20
    lens = [18, 21, -1, 5, 5, 5, 5]
    count = [3, 0, 1, 5, -1, 2, 2]
    path = [[0, 1, 2, 3]] * 5 + [[0, 4, -1, -1], [0, 2, -1, -1]]
    x = inputs(torch.float16, B, n, Hk, Hk, D, cap, [0] * B, [tree(n, 2)] * B, seed=13)
    before = x["k_cache"].clone()
    new = cc.draft_commit(x["k_cache"], x["v_cache"], i32(lens), x["k_new"], x["v_new"], i32(path), i32(count))
    assert new.tolist() == lens[:6] + [7]
    assert torch.equal(x["k_cache"][:6], before[:6]) and not torch.equal(x["k_cache"][6], before[6])
    acc = torch.ones(B, Hk, cap, device="cuda")
    cc.draft_accumulate(x["q"], torch.zeros(B, n, Hk, device="cuda"), x["k_cache"], i32(lens), i32(path), i32(count), acc)
    assert (acc[:6] == 1).all() and not (acc[6] == 1).all()
    torch.cuda.synchronize()
    with pytest.raises(eng.CKKSError) as e:
        cc.Synchronize()
    assert e.value.code == 7 and "6 sequence" in str(e.value)
    cc.Synchronize()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 1, 12, 12, 64, 128, [103], [1]), (3, 9, 8, 2, 128, 700, [500, 0, 691], [4, 9, 5]),
                                   (2, 64, 4, 4, 64, 400, [129, 336], [64, 3]), (2, 5, 6, 3, 80, 300, [290, 128], [5, 0]),
                                   (1, 3, 2, 1, 33, 70, [60], [2]), (1, 2, 8, 1, 256, 3000, [2998], [2]),
                                   (2, 16, 16, 2, 96, 260, [240, 3], [16, 16]),
                                   (3, 4, 4, 2, 8, 620000, [300000, 0, 619996], [3, 0, 4]),  # divided as a list
                                   (1, 3, 2, 1, 8, 1500000, [1499990], [2])])
def test_accumulate(cc, dtype, shape):
    """A weight is exp of a score off by (D + 8) 2^-24 S and an lse off by
    2^-24 of itself; the sum over the rows adds their number of roundings."""
    B, n, Hq, Hk, D, cap, lens, count = shape
    x = inputs(dtype, B, n, Hq, Hk, D, cap, lens, [tree(n, 1)] * B, seed=14)
    path = i32([list(range(n))] * B)
    _, lse = cc.draft_attention(**x)
    cc.draft_commit(x["k_cache"], x["v_cache"], x["lens"], x["k_new"], x["v_new"], path, i32(count))
    acc = torch.rand(B, Hk, cap, device="cuda")
    args = (f64(x["q"]), f64(lse), f64(x["k_cache"]), lens, path.cpu().numpy(), count)
    want = ref.accumulate(*args, f64(acc), D ** -0.5)
    got = cc.draft_accumulate(x["q"], lse, x["k_cache"], x["lens"], path, i32(count), acc)
    assert got is acc
    S = np.abs(f64(x["q"])).max(-1).max() * np.abs(f64(x["k_cache"])).sum(-1).max() * D ** -0.5
    room = 2.0 ** -23 * ((D + 8) * S + np.abs(f64(lse)[np.isfinite(f64(lse))]).max() + n * Hq // Hk + 4) * want
    assert (np.abs(f64(acc) - want) <= room).all()
    for b in range(B):  # a chain's rows give each head as much weight as there are rows
        if count[b] and lens[b] + count[b] <= cap:
            gain = f64(acc)[b, :, :lens[b] + count[b]].sum() - f64(acc)[b].sum()
            assert np.isfinite(gain)
    cc.Synchronize()


@pytest.mark.parametrize("dtype", TYPES)
def test_accumulated_weight_adds_up(cc, dtype):
    """The rows of a chain sum to 1 each: a head's weights grow by the number
    of accepted rows, to 2^-10 of it."""
    x = inputs(dtype, 2, 6, 8, 2, 64, 1000, [900, 17], [tree(6, 1)] * 2, seed=15)
    _, lse = cc.draft_attention(**x)
    path, count = i32([list(range(6))] * 2), i32([6, 4])
    cc.draft_commit(x["k_cache"], x["v_cache"], x["lens"], x["k_new"], x["v_new"], path, count)
    acc = cc.draft_accumulate(x["q"], lse, x["k_cache"], x["lens"], path, count, torch.zeros(2, 2, 1000, device="cuda"))
    want = np.array([[6 * 4.0] * 2, [4 * 4.0] * 2])
    assert (np.abs(f64(acc).sum(-1) - want) <= 2.0 ** -10 * want).all()


def check_evict(x, acc, budget, recent, got, before):
    k2, v2, a2, index, new = got
    lens = x["lens"].tolist()
    for b, m in enumerate(lens):
        m = min(max(m, 0), acc.shape[2])
        for h in range(acc.shape[1]):
            rows = ref.keep(f64(acc[b, h]), m, budget, recent)
            a = len(rows)
            assert index[b, h].tolist() == list(rows) + [-1] * (budget - a)
            pick = torch.tensor(rows, device="cuda", dtype=torch.long)
            for out, src, old in ((k2, x["k_cache"], before[0]), (v2, x["v_cache"], before[1]), (a2, acc, before[2])):
                assert torch.equal(out[b, h, :a].nan_to_num(), src[b, h, pick].nan_to_num())
                assert torch.equal(out[b, h, a:], old[b, h, a:])
        assert int(new[b]) == min(m, budget)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 3, 64, 2100, [2100], 1000, 100), (4, 2, 128, 300, [300, 0, 64, 65], 64, 8),
                                   (2, 2, 33, 90, [90, 41], 41, 41), (1, 1, 80, 50, [50], 1, 0), (1, 1, 64, 50, [50], 1, 1),
                                   (2, 1, 1, 5000, [5000, 4097], 4096, 5), (1, 2, 96, 70000, [70000], 9000, 300),
                                   (3, 2, 40, 30, [40, -4, 30], 29, 3), (1, 2, 16, 12000, [12000], 5000, 100),
                                   (2, 1, 8, 200000, [200000, 131073], 40000, 0)])
def test_evict(cc, dtype, shape):
    B, Hk, D, cap, lens, budget, recent = shape
    x = inputs(dtype, B, 1, Hk, Hk, D, cap, lens, [[-1]] * B, seed=16)
    acc = torch.exp(2 * torch.randn(B, Hk, cap, device="cuda", generator=torch.Generator(device="cuda").manual_seed(17)))
    rows = budget + 5
    out = (torch.full((B, Hk, rows, D), 7.0, dtype=dtype, device="cuda"),
           torch.full((B, Hk, rows, D), 8.0, dtype=dtype, device="cuda"), torch.full((B, Hk, rows), 9.0, device="cuda"))
    before = [t.clone() for t in out]
    check_evict(x, acc, budget, recent, cc.draft_evict(x["k_cache"], x["v_cache"], acc, x["lens"], budget, recent, out),
                before)
    fresh = cc.draft_evict(x["k_cache"], x["v_cache"], acc, x["lens"], budget, recent)
    check_evict(x, acc, budget, recent, fresh, [torch.zeros_like(t) for t in fresh[:3]])


@pytest.mark.parametrize("kind", ["equal", "two", "zeros", "special", "close", "negative"])
def test_evict_ties(cc, kind):
    """Equal weights go to the lower index; -0 equals 0; NaN goes last."""
    cap, budget, recent = 3000, 1100, 50
    g = torch.Generator(device="cuda").manual_seed(18)
    acc = torch.ones(2, 2, cap, device="cuda")
    if kind == "two":
        acc = torch.randint(0, 2, (2, 2, cap), generator=g, device="cuda").float()
    elif kind == "zeros":
        acc = torch.where(torch.rand(2, 2, cap, generator=g, device="cuda") < 0.5, 0.0, -0.0)
    elif kind == "special":
        acc = torch.rand(2, 2, cap, generator=g, device="cuda")
        acc[:, :, ::3] = float("nan")
        acc[:, :, 1::5] = float("inf")
        acc[:, :, 2::7] = float("-inf")
    elif kind == "close":  # neighbouring floats: the last bits decide
        acc = (torch.randint(0, 300, (2, 2, cap), generator=g, device="cuda", dtype=torch.int32) + 0x3F800000).view(torch.float32)
    elif kind == "negative":
        acc = -torch.rand(2, 2, cap, generator=g, device="cuda").round(decimals=2)
    x = inputs(torch.bfloat16, 2, 1, 2, 2, 64, cap, [cap, cap - 1], [[-1]] * 2, seed=19)
    for b, r in ((budget, recent), (1, 0), (cap - 2, 0), (cap - 2, cap - 2), (2100, 0)):
        got = cc.draft_evict(x["k_cache"], x["v_cache"], acc, x["lens"], b, r)
        check_evict(x, acc, b, r, got, [torch.zeros_like(t) for t in got[:3]])


def test_cache_strides_and_streams(cc):
    """Head-interleaved caches and weights in larger buffers, on another
    stream and in a graph."""
    x = inputs(torch.bfloat16, 2, 3, 4, 2, 64, 500, [480, 200], [tree(3, 1)] * 2, seed=20)
    mixed = {k: x[k].transpose(1, 2).contiguous().transpose(1, 2) for k in ("k_cache", "v_cache")}
    wide = torch.zeros(2, 2, 700, device="cuda")
    path, count = i32([[0, 1, 2]] * 2), i32([3, 1])
    _, lse = cc.draft_attention(**x)
    a = torch.zeros(2, 2, 500, device="cuda")

    def step(k, v, acc):
        new = cc.draft_commit(k, v, x["lens"], x["k_new"], x["v_new"], path, count)
        cc.draft_accumulate(x["q"], lse, k, x["lens"], path, count, acc)
        return cc.draft_evict(k, v, acc, new, 100, 10)

    want = step(x["k_cache"], x["v_cache"], a)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = step(mixed["k_cache"], mixed["v_cache"], wide[:, :, 100:600])
    s.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(want, got))
    assert torch.equal(wide[:, :, 100:600], a) and not wide[:, :, :100].any() and not wide[:, :, 600:].any()
    odd = torch.zeros(2, 2, 700, device="cuda")  # weights off every wide boundary
    got = step(mixed["k_cache"], mixed["v_cache"], odd[:, :, 101:601])
    assert all(torch.equal(p, q) for p, q in zip(want, got))
    g = torch.cuda.CUDAGraph()
    a.zero_()
    with torch.cuda.graph(g):
        out = step(x["k_cache"], x["v_cache"], a)
    a.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(want, out))


# ---- refusals at the C ABI ------------------------------------------------------------

def test_refusals(cc):
    x = inputs(torch.bfloat16, 2, 3, 4, 2, 64, 50, [50, 20], [tree(3, 1)] * 2)
    with pytest.raises(eng.CKKSError):
        cc.draft_attention(**(dict(x) | {"q": torch.zeros(2, 3, 3, 64, dtype=torch.bfloat16, device="cuda")}))
    with pytest.raises(eng.CKKSError):
        cc.draft_attention(**x, scale=float("nan"))
    y = inputs(torch.bfloat16, 1, 65, 2, 2, 64, 50, [50], [tree(65, 1)])
    with pytest.raises(eng.CKKSError):
        cc.draft_attention(**y)
    y = inputs(torch.bfloat16, 1, 2, 2, 2, 257, 50, [50], [tree(2, 1)])
    with pytest.raises(eng.CKKSError):
        cc.draft_attention(**y)
    with pytest.raises(ValueError):
        cc.draft_attention(**(dict(x) | {"lens": x["lens"].cpu()}))
    acc = torch.zeros(2, 2, 50, device="cuda")
    for budget, recent in ((0, 0), (5, 6), (5, -1)):
        with pytest.raises(ValueError):
            cc.draft_evict(x["k_cache"], x["v_cache"], acc, x["lens"], budget, recent)
    with pytest.raises(eng.CKKSError) as e:  # in place
        cc.draft_evict(x["k_cache"], x["v_cache"], acc, x["lens"], 40, 5, out=(x["k_cache"], x["v_cache"], acc))
    assert "overlaps" in str(e.value)
    path, count = i32([[0, 1, 2]] * 2), i32([1, 1])
    with pytest.raises(eng.CKKSError, match="overlap the cache"):
        new = x["k_cache"][:, :, 40:43].transpose(1, 2)
        cc.draft_commit(x["k_cache"], x["v_cache"], x["lens"], new, x["v_new"], path, count)
    with pytest.raises(eng.CKKSError):
        cc.draft_accumulate(x["q"], torch.zeros(2, 3, 4, device="cuda"), x["k_cache"], x["lens"], path, count, acc, 1e39)
    v = verify_inputs(2, 3, 10, 1, torch.float32, torch.float32, 1)
    with pytest.raises(eng.CKKSError):  # a tree without nodes
        cc.draft_verify(v["target"][:, :1], v["draft"][:, :1], v["tokens"][:, :0], v["parents"][:, :0],
                        v["uniforms"][:, :1].contiguous())
    cc.Synchronize()


class Rows(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p)] + [(n, ctypes.c_int64) for n in ("batch", "head", "row")]


class AttentionArgs(ctypes.Structure):
    """ckks_draft_attention_args of include/ckks_b200.h."""
    _fields_ = ([(n, ctypes.c_int32) for n in ("dtype", "batch", "q_heads", "kv_heads", "head_dim", "nodes", "capacity",
                                               "reserved")] + [("scale", ctypes.c_double)]
                + [(n, Rows) for n in ("q", "k_cache", "v_cache", "k_new", "v_new", "out")]
                + [(n, ctypes.c_void_p) for n in ("lens", "parents", "lse", "workspace")]
                + [("workspace_bytes", ctypes.c_size_t)])


def test_refused_structs(cc):
    """What torch tensors never hold, at the C entry points."""
    lib, buf = eng.lib(), torch.zeros(4096, device="cuda")
    at = buf.data_ptr()

    def attention(**change):
        f = dict(dtype=0, batch=1, q_heads=2, kv_heads=1, head_dim=16, nodes=2, capacity=4, reserved=0, scale=1.0,
                 lens=at, parents=at, lse=at, workspace=at, workspace_bytes=1 << 14)
        f |= {n: Rows(at, 64, 16, 16) for n in ("q", "k_cache", "v_cache", "k_new", "v_new", "out")}
        a = AttentionArgs(**(f | change))
        return lib.ckks_draft_attention(cc.h, ctypes.byref(a), None)

    assert attention(batch=0) == 0
    for change in (dict(dtype=3), dict(dtype=9), dict(dtype=-1), dict(batch=-1), dict(q_heads=3, kv_heads=2),
                   dict(q_heads=0), dict(kv_heads=0), dict(head_dim=0), dict(head_dim=257), dict(nodes=0),
                   dict(nodes=65), dict(capacity=-1), dict(capacity=1 << 30), dict(reserved=1),
                   dict(scale=float("inf")), dict(q=Rows(0, 64, 16, 16)), dict(q=Rows(at + 1, 64, 16, 16)),
                   dict(k_cache=Rows(at, -64, 16, 16)), dict(out=Rows(0, 64, 16, 16)), dict(lens=0), dict(lens=at + 2),
                   dict(parents=0), dict(lse=0), dict(workspace=at + 4), dict(batch=1 << 30, q_heads=64, kv_heads=1)):
        assert attention(**change) == 1, change
        assert lib.ckks_last_error()
    assert attention(nodes=64, q_heads=8, capacity=4000, workspace_bytes=16) == 1  # too small
    assert lib.ckks_draft_attention(cc.h, None, None) == 1
    cc.Synchronize()
