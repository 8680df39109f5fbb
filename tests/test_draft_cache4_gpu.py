"""Caches in 4 bits on the GPU: rows written, committed and read back, bit for
bit against tests/prompt_reference.py, and attention over them against the
float64 definition of draft_reference.py on the values that they hold.

Bounds as in tests/test_draft_gpu.py, and half of the smallest steps: one in
nine values of a 4-bit cache is 0, so a row whose heaviest keys have the value 0
has results far below its weights.  A float16 result below 2^-14 is off by up
to 2^-25 whatever its size (half a step of 2^-24).  With 16-bit queries, of
either type, the weights are float16 numbers: steps of 2^-24 where the largest
is 2^7 or more, so each is off by up to 2^-25 / 2^7 = 2^-32 of the largest,
times |v|, and their sum is at least the largest.  The other smallest steps are
below 1e-30."""

import ctypes

import numpy as np
import pytest

import draft_reference
import prompt_reference as ref

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import private_genomic_dnagpt_b200 as eng  # noqa: E402
from private_genomic_dnagpt_b200 import drafting  # noqa: E402

import test_draft_gpu as base  # noqa: E402
from test_draft_gpu import HALF, SHAPES, TYPES, f64, i32, tree  # noqa: E402
from test_draft_prompt_gpu import packed  # noqa: E402


@pytest.fixture(scope="module")
def cc():
    return eng.GenCryptoContext(eng.CCParams(ring_dim_log=10, limbs=3, dnum=1, seed=3))


def cuda8(rows):
    return torch.from_numpy(np.ascontiguousarray(rows)).cuda()


def awkward(dtype, rows, D, seed):
    """Rows at the places where rounding turns: middles between two numbers of
    a scale and between two scales, their neighbours, the ends of the range,
    zeros of either sign."""
    rng = np.random.default_rng(seed)
    s = ref.SCALES[rng.integers(1, len(ref.SCALES), (rows, -(-D // 16)))].repeat(16, -1)[:, :D]
    x = s * rng.choice([0.25, 0.5, 0.75, 1.0, 1.25, 1.5, 1.75, 2.0, 2.5, 3.0, 3.5, 4.0, 5.0, 6.0, 6.2], (rows, D))
    x[:, 0] = 6 * s[:, 0]
    x *= rng.choice([1.0, -1.0], (rows, D))
    x[rng.random((rows, D)) < 0.05] = 0.0
    x[rng.random((rows, D)) < 0.05] *= -0.0
    t = torch.from_numpy(x).to(dtype)
    if dtype == torch.float32:  # one step to either side
        bits = t.view(torch.int32)
        bits += torch.from_numpy(rng.integers(-1, 2, (rows, D)).astype(np.int32)) * (t != 0)
    t[-4] *= 1e-6
    t[-3] = torch.from_numpy(rng.choice([61440.0, 6e4, 65504.0, -65504.0, 1.0], D)).to(dtype)
    t[-2] = 0.0
    if dtype != torch.float16:
        t[-1] *= 1e30
    return t.cuda()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 128, 80, 40, 33, 1, 256, 100, 16])
def test_written_rows_bit_for_bit(cc, dtype, D):
    assert drafting.row4_bytes(D) == ref.row_bytes(D)
    T, H, cap = 120, 3, 130
    k = awkward(dtype, T * H, D, 20).view(T, H, D)
    v = torch.randn(T, H, D, device="cuda").to(dtype)
    starts, lens = packed([50, 0, 69], 1), [7, 2, 61]
    caches = [torch.full((3, H, cap, ref.row_bytes(D)), 0x11, dtype=torch.uint8, device="cuda") for _ in range(2)]
    want = [ref.fill(c.cpu().numpy(), lens, ref.pack(f64(x)), starts) for c, x in zip(caches, (k, v))]
    got = cc.draft_fill4(*caches, i32(lens), k, v, i32(starts))
    assert got.tolist() == [57, 2, 130] == want[0][1].tolist()
    for c, w in zip(caches, want):
        assert np.array_equal(c.cpu().numpy(), w[0])
    for t in TYPES:
        for c, w in zip(caches, want):
            back = f64(cc.draft_read4(c, got, D, t))
            values = ref.unpack(w[0], D)
            for b, m in enumerate(got.tolist()):
                assert np.array_equal(back[b, :, :m], values[b, :, :m]) and not back[b, :, m:].any()
    cc.Synchronize()


@pytest.mark.parametrize("dtype", TYPES)
def test_every_number_of_every_scale(cc, dtype):
    """What a row can hold is written and read back unchanged, 16 numbers of
    each scale that has an exact 6 in the group."""
    x = ref.SCALES[1:, None] * np.concatenate([ref.VALUES, -ref.VALUES])
    k = torch.from_numpy(x).to(dtype).cuda()[:, None]
    n = len(x)
    cache = torch.zeros(1, 1, n, 12, dtype=torch.uint8, device="cuda"), torch.zeros(1, 1, n, 12, dtype=torch.uint8, device="cuda")
    cc.draft_fill4(*cache, i32([0]), k, k, i32([0, n]))
    assert np.array_equal(f64(cc.draft_read4(cache[1], i32([n]), 16, dtype))[0, 0], x)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_groups_that_are_not_finite(cc, dtype, bad):
    k = torch.randn(5, 2, 40, device="cuda").to(dtype)
    k[2, 1, 17] = bad
    cache = [torch.zeros(1, 2, 6, ref.row_bytes(40), dtype=torch.uint8, device="cuda") for _ in range(2)]
    lens = cc.draft_fill4(*cache, i32([0]), k, k, i32([0, 5]))
    for t in TYPES:
        back = cc.draft_read4(cache[0], lens, 40, t)[0]
        spoiled = torch.isnan(back)
        assert spoiled[1, 2, 16:32].all() and int(spoiled.sum()) == 16


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 33, 256])
def test_commit4(cc, dtype, D):
    """The accepted nodes of each sequence, as ``draft_commit`` takes them."""
    B, n, H, cap = 5, 9, 2, 40
    k, v = (awkward(dtype, B * n * H, D, s).view(B, n, H, D) for s in (21, 22))
    path = np.full((B, n), -1)
    path[0, :3], path[1, :9], path[2, :2], path[3, :1], path[4, :2] = [0, 4, 8], range(9), [3, 9], [5], [1, 2]
    lens, count = [0, 31, 4, 40, 12], [3, 9, 2, 1, 0]
    caches = [torch.full((B, H, cap, ref.row_bytes(D)), 7, dtype=torch.uint8, device="cuda") for _ in range(2)]
    want = [c.cpu().numpy().copy() for c in caches]
    for b in (0, 1):
        for j in range(count[b]):
            for w, x in zip(want, (k, v)):
                w[b, :, lens[b] + j] = ref.pack(f64(x[b, path[b, j]]))
    got = cc.draft_commit4(*caches, i32(lens), k, v, i32(path), i32(count))
    assert got.tolist() == [3, 40, 4, 40, 12]  # a node that is not there, and a full cache
    for c, w in zip(caches, want):
        assert np.array_equal(c.cpu().numpy(), w)
    with pytest.raises(eng.CKKSError, match=r"2 sequence\(s\) left unchanged"):
        cc.Synchronize()


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_of_caches_and_rows(cc, dtype):
    """Heads and rows in other orders, rows apart, sources off every wide
    boundary, an output that torch lays out."""
    T, H, D, cap = 70, 2, 64, 80
    k, v = (torch.randn(T, H, D, device="cuda").to(dtype) for _ in range(2))
    R = ref.row_bytes(D)
    plain = [torch.zeros(2, H, cap, R, dtype=torch.uint8, device="cuda") for _ in range(2)]
    lens = cc.draft_fill4(*plain, i32([0, 3]), k, v, i32([0, 40, 70]))
    inner = torch.zeros(2, cap, H, R, dtype=torch.uint8, device="cuda").transpose(1, 2)
    apart = torch.zeros(2, H, cap, R + 4, dtype=torch.uint8, device="cuda")[..., :R]
    flat = torch.zeros(k.numel() + 1, dtype=dtype, device="cuda")
    flat[1:] = k.reshape(-1)
    got = cc.draft_fill4(inner, apart, i32([0, 3]), flat[1:].view(T, H, D), v.transpose(0, 1).contiguous().transpose(0, 1),
                         i32([0, 40, 70]))
    assert torch.equal(got, lens) and torch.equal(inner, plain[0]) and torch.equal(apart, plain[1])
    assert not torch.as_strided(apart, (2, H, cap, 4), apart.stride(), R).any()
    for a, b in zip((inner, apart), plain):
        assert torch.equal(cc.draft_read4(a, lens, D, dtype), cc.draft_read4(b, lens, D, dtype))


def check_attention(x, out, lse, scale=None):
    q, v = f64(x["q"]), f64(x["v_cache"])
    D = q.shape[3]
    scale = D ** -0.5 if scale is None else scale
    want, wlse, mag, big, keys = draft_reference.attention(q, f64(x["k_cache"]), v, x["lens"].cpu().numpy(),
                                                           f64(x["k_new"]), f64(x["v_new"]), x["parents"].cpu().numpy(),
                                                           scale)
    got, glse = f64(out), f64(lse)
    noise = 2.0 ** -23 * ((D + 8) * big + keys + 8)
    room = (2 * HALF[x["q"].dtype] + noise)[..., None] * mag + 1e-30
    if x["q"].dtype != torch.float32:
        top = max(np.abs(v).max(initial=0.0), np.abs(f64(x["v_new"])).max())
        room += 2.0 ** -32 * top * keys[..., None]
    if x["q"].dtype == torch.float16:
        room += 2.0 ** -25
    assert np.isfinite(want).all() and np.isfinite(got).all()
    worst = (np.abs(got - want) / room).max()
    assert worst <= 1.0, f"out: {worst:.3g} times the bound"
    seen = keys > 0
    assert np.array_equal(glse == -np.inf, ~seen)
    assert (np.abs(glse[seen] - wlse[seen]) <= (0.5 * noise + 2.0 ** -22 * (1 + np.abs(wlse)))[seen]).all()
    assert not got[~seen].any()


def quantised(x):
    """``inputs`` of a tree with its caches packed; and the same with the
    values that they hold, for the reference."""
    y, z = dict(x), dict(x)
    for name in ("k_cache", "v_cache"):
        rows = ref.pack(f64(x[name]))
        y[name], z[name] = cuda8(rows), torch.from_numpy(ref.unpack(rows, x[name].shape[-1])).cuda()
    return y, z


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_attention4(cc, dtype, shape):
    B, n, Hq, Hk, D, cap, lens, branch, pad = shape
    x = base.inputs(dtype, B, n, Hq, Hk, D, cap, lens, [tree(n, branch, pad if b == B - 1 else 0) for b in range(B)])
    y, z = quantised(x)
    check_attention(z, *cc.draft_attention4(**y))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(2, 13, 8, 2, 128, 9000, [8999, 4097], 3), (1, 1, 4, 4, 64, 20000, [19999], 1),
                                   (1, 40, 4, 1, 64, 5000, [4999], 2), (2, 1, 8, 1, 128, 30001, [30001, 257], 1),
                                   (2, 21, 4, 1, 256, 9000, [8999, 4097], 3)])
def test_attention4_over_long_caches(cc, dtype, shape):
    B, n, Hq, Hk, D, cap, lens, branch = shape
    x = base.inputs(dtype, B, n, Hq, Hk, D, cap, lens, [tree(n, branch)] * B, seed=1)
    y, z = quantised(x)
    check_attention(z, *cc.draft_attention4(**y))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 128, 200])
@pytest.mark.parametrize("n", [1, 6, 50])
def test_attention4_sharp_rows(cc, dtype, D, n):
    x = base.inputs(dtype, 2, n, 4, 2, D, 600, [600, 321], [tree(n, 2)] * 2, seed=2, spread=6.0)
    y, z = quantised(x)
    check_attention(z, *cc.draft_attention4(**y))
    for scale in (0.5, -0.01, 0.0):
        check_attention(z, *cc.draft_attention4(**y, scale=scale), scale=scale)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 128, 40, 256])
@pytest.mark.parametrize("n", [1, 10])
def test_attention4_ignores_what_is_masked(cc, dtype, D, n):
    """Rows behind the length are NaN, whatever the codes, and so are padding nodes."""
    lens, pad = [130, 0, 257], 3 if n > 3 else 0
    x = base.inputs(dtype, 3, n, 4, 2, D, 300, lens, [tree(n, 2, pad)] * 3, seed=4)
    y, _ = quantised(x)
    clean = cc.draft_attention4(**y)
    for b, m in enumerate(lens):
        y["k_cache"][b, :, m:] = 0xFC
        y["v_cache"][b, :, m:] = 0xFC
    for name in ("k_new", "v_new", "q"):
        y[name][:, n - pad:] = float("nan")
    got = cc.draft_attention4(**y)
    assert torch.equal(clean[0], got[0]) and torch.equal(clean[1], got[1])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 128, 40, 256])
@pytest.mark.parametrize("G", [1, 4])
def test_attention4_keeps_siblings_apart(cc, dtype, D, G):
    parents = [-1, -1, 0, 0, 1, 1, 4]
    x = base.inputs(dtype, 2, 7, 2 * G, 2, D, 200, [190, 0], [parents] * 2, seed=5)
    y, _ = quantised(x)
    clean = f64(cc.draft_attention4(**y)[0])
    y["k_new"][:, 1] = float("nan")
    y["v_new"][:, 1] = float("nan")
    y["v_new"][:, 3] = float("inf")
    got, lse = (f64(t) for t in cc.draft_attention4(**y))
    for i in (0, 2):
        assert np.array_equal(got[:, i], clean[:, i])
    for i in (1, 4, 5, 6):
        assert np.isnan(got[:, i]).all() and np.isnan(lse[:, i]).all()
    assert (got[:, 3] == np.inf).all() and np.isfinite(lse[:, 3]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D,G", [(64, 1), (128, 4), (40, 2)])
@pytest.mark.parametrize("at", [0, 77, 2500, 4999])
def test_attention4_shows_groups_that_are_not_finite(cc, dtype, D, G, at):
    """A value that is no number spoils its elements of every row, also where
    its weight is exp(-1000) of the others'; a key spoils the row."""
    x = base.inputs(dtype, 1, 3, G, 1, D, 5000, [5000], [tree(3, 1)], seed=40)
    for name in ("q", "k_cache", "k_new"):
        x[name][..., 0] = 0.0
    x["q"][..., 0] = D ** 0.5
    x["k_cache"][:, :, at, 0] = -1000.0
    y, _ = quantised(x)
    G4 = -(-D // 16)
    y["v_cache"][:, :, at, 8 * G4 + 1] = 0xFC
    got = f64(cc.draft_attention4(**y)[0])
    assert not np.isfinite(got[..., 16:32]).any()
    assert np.isfinite(got[..., :16]).all() and np.isfinite(got[..., 32:]).all()
    y["k_cache"][:, :, at, 8 * G4] = 0xFC
    assert np.isnan(f64(cc.draft_attention4(**y)[0])).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 12])
def test_attention4_strides(cc, dtype, n):
    x = base.inputs(dtype, 2, n, 4, 2, 64, 208, [200, 111], [tree(n, 2)] * 2, seed=8)
    y, z = quantised(x)
    want = cc.draft_attention4(**y)
    a = dict(y)
    a["q"] = y["q"].transpose(1, 2).contiguous().transpose(1, 2)
    a["k_new"] = y["k_new"].transpose(1, 2).contiguous().transpose(1, 2)
    got = cc.draft_attention4(**a)
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
    b = dict(y)
    b["k_cache"] = y["k_cache"].transpose(1, 2).contiguous().transpose(1, 2)
    wide = torch.zeros(2, 2, 208, 40, dtype=torch.uint8, device="cuda")
    wide[..., :36] = y["v_cache"]
    b["v_cache"] = wide[..., :36]
    check_attention(z, *cc.draft_attention4(**b))
    odd = torch.zeros(y["k_cache"].numel() + 4, dtype=torch.uint8, device="cuda")  # on a 4-byte boundary only
    odd[4:] = y["k_cache"].reshape(-1)
    check_attention(z, *cc.draft_attention4(**(y | {"k_cache": odd[4:].view(y["k_cache"].shape)})))
    for name in ("q", "k_new", "v_new"):
        flat = torch.zeros(x[name].numel() + 1, dtype=dtype, device="cuda")
        flat[1:] = x[name].reshape(-1)
        check_attention(z, *cc.draft_attention4(**(y | {name: flat[1:].view(x[name].shape)})))
    one = y | {"k_cache": y["k_cache"][:1].expand_as(y["k_cache"])}
    check_attention(z | {"k_cache": z["k_cache"][:1].expand_as(z["k_cache"])}, *cc.draft_attention4(**one))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_offsets_past_32_bits(cc, dtype):
    """Rows and heads far apart: the last ones lie past 2^32 bytes."""
    cap, R = 70, ref.row_bytes(64)
    store = torch.empty(5 << 30, dtype=torch.uint8, device="cuda")
    x = base.inputs(dtype, 1, 3, 2, 2, 64, cap, [cap], [tree(3, 1)], seed=9)
    y, z = quantised(x)
    for step, head in ((1 << 26, 64), (R, (4 << 30) + 16)):
        for name, at in (("k_cache", 0), ("v_cache", 8192)):
            view = torch.as_strided(store, (1, 2, cap, R), (R, head, step, 1), at)
            view.copy_(y[name])
            a = y | {name: view}
            check_attention(z, *cc.draft_attention4(**a))
            assert np.array_equal(f64(cc.draft_read4(view, i32([cap]), 64, dtype)), f64(z[name]))


@pytest.mark.parametrize("dtype,D,n", [(torch.bfloat16, 64, 5), (torch.float16, 128, 21), (torch.float32, 64, 1),
                                       (torch.bfloat16, 128, 1)])
def test_attention4_repeats_streams_and_graphs(cc, dtype, D, n):
    xs = [base.inputs(dtype, 2, n, 8, 2, D, 6000, [5999 - s, 3000], [tree(n, 2)] * 2, seed=11 + s) for s in range(2)]
    xs = [quantised(x)[0] for x in xs]
    want = [cc.draft_attention4(**x) for x in xs]
    again = cc.draft_attention4(**xs[0])
    assert torch.equal(again[0], want[0][0]) and torch.equal(again[1], want[0][1])
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = cc.draft_attention4(**xs[0])
    s.synchronize()
    assert torch.equal(got[0], want[0][0])
    graphs, outs = [], []
    for x in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(cc.draft_attention4(**x))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    for _ in range(10):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert torch.equal(o[0], w[0]) and torch.equal(o[1], w[1])


def test_lengths_and_parents_out_of_range(cc):
    x = base.inputs(torch.float16, 3, 2, 2, 2, 64, 96, [500, -3, 96], [[-1, 1], [-7, 0], [-1, 0]], seed=7)
    y, z = quantised(x)
    check_attention(z, *cc.draft_attention4(**y))


def test_one_row_of_each_size(cc):
    """Empty batches and caches without rows."""
    x = base.inputs(torch.bfloat16, 0, 3, 2, 2, 64, 10, np.zeros(0), np.zeros((0, 3)))
    empty = torch.zeros(0, 2, 10, 36, dtype=torch.uint8, device="cuda")
    out, lse = cc.draft_attention4(**(x | {"k_cache": empty, "v_cache": empty}))
    assert out.shape == (0, 3, 2, 64) and lse.shape == (0, 3, 2)
    none = torch.zeros(2, 2, 0, 36, dtype=torch.uint8, device="cuda")
    assert cc.draft_read4(none, i32([0, 0]), 64, torch.bfloat16).shape == (2, 2, 0, 64)
    assert cc.draft_read4(empty, i32([]), 64, torch.bfloat16).shape == (0, 2, 10, 64)
    k = torch.zeros(3, 2, 64, device="cuda")
    assert cc.draft_fill4(none, none.clone(), i32([0, 0]), k[:0], k[:0], i32([0, 0, 0])).tolist() == [0, 0]
    cc.Synchronize()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,D", [(1, 64), (9, 128), (40, 256)])
def test_attention4_of_queries_of_any_size(cc, dtype, n, D):
    """Queries times 2^60 or 2^-60, with the scale that takes it back, give the
    same bits; rows of a tree may differ in size."""
    x = base.inputs(dtype, 2, n, 4, 2, D, 500, [500, 129], [tree(n, 2)] * 2, seed=30)
    y, z = quantised(x)
    want = cc.draft_attention4(**y)
    for power in (2.0 ** 60, 2.0 ** -60):
        got = cc.draft_attention4(**(y | {"q": y["q"] * power}), scale=D ** -0.5 / power)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    sizes = torch.tensor([10.0 ** (i % 5 - 3) for i in range(n)], device="cuda")[:, None, None]
    q = (y["q"].float() * sizes).to(dtype)
    check_attention(z | {"q": q}, *cc.draft_attention4(**(y | {"q": q})))


@pytest.mark.parametrize("dtype", TYPES)
def test_attention4_from_two_threads(cc, dtype):
    """Calls of other sizes at the same time from two host threads."""
    import threading
    xs = [quantised(base.inputs(dtype, 1, n, 4, 4, D, 700, [650], [tree(n, 2)], seed=31))[0] for n, D in ((1, 64), (20, 128))]
    want = [cc.draft_attention4(**x) for x in xs]
    torch.cuda.synchronize()
    wrong = []

    def calls(x, w):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(50):
                got = cc.draft_attention4(**x)
                torch.cuda.current_stream().synchronize()
                if not (torch.equal(got[0], w[0]) and torch.equal(got[1], w[1])):
                    wrong.append(1)

    threads = [threading.Thread(target=calls, args=a) for a in zip(xs, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
    cc.Synchronize()


def test_captured_run_of_prompt_fill_and_trees(cc):
    """A whole run captured into one graph and replayed over other inputs:
    prompt, its rows into 4 bits, a tree over them, its commit, a second tree."""
    g = torch.Generator(device="cuda").manual_seed(32)
    normal = lambda *s: torch.randn(*s, generator=g, device="cuda").to(torch.bfloat16)  # noqa: E731
    H, D, T, n = 4, 64, 300, 6
    q, k, v = normal(T, H, D), normal(T, H, D), normal(T, H, D)
    qt, kt, vt = normal(2, n, H, D), normal(2, n, H, D), normal(2, n, H, D)
    starts, parents, path, count = i32([0, 120, 300]), i32([tree(n, 2)] * 2), i32([[0, 2, -1, -1, -1, -1]] * 2), i32([2, 1])

    def run():
        caches = [torch.zeros(2, H, 256, drafting.row4_bytes(D), dtype=torch.uint8, device="cuda") for _ in range(2)]
        out, lse = cc.draft_prompt(q, k, v, starts)
        lens = cc.draft_fill4(*caches, i32([0, 0]) if not torch.cuda.is_current_stream_capturing() else zero, k, v, starts)
        tree_out, _ = cc.draft_attention4(qt, *caches, lens, kt, vt, parents)
        lens = cc.draft_commit4(*caches, lens, kt, vt, path, count)
        again, _ = cc.draft_attention4(qt, *caches, lens, kt, vt, parents)
        return out, lse, tree_out, again, lens, cc.draft_read4(caches[0], lens, D, torch.bfloat16)

    zero = i32([0, 0])
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    for t in (q, k, v, qt, kt, vt):
        t.copy_(normal(*t.shape))
    starts.copy_(i32([0, 200, 290]))
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, run()):
        assert torch.equal(a, b)
    assert got[4].tolist() == [202, 91]
    cc.Synchronize()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,D", [(1, 64), (9, 128), (40, 256)])
@pytest.mark.parametrize("power", [8, 13, 20, 24, 40, 120])
def test_attention4_of_rows_with_elements_far_apart(cc, dtype, n, D, power):
    """The keys are 0 where a query's elements are 2^power times its others,
    so that the scores consist of the others; then keys and queries scaled
    oppositely by 2^13, so that both parts weigh the same.  Every product of a
    cached value and an element has its place in a 32-bit sum, so the bounds are
    those of every other row."""
    if dtype == torch.float16 and power > 8:
        power = 13  # of 16
    x = base.inputs(dtype, 2, n, 4, 2, D, 500, [500, 129], [tree(n, 2)] * 2, seed=50)
    big = dict(x) | {name: x[name].clone() for name in ("q", "k_cache", "k_new")}
    big["q"][..., :16] *= 2.0 ** power
    for name in ("k_cache", "k_new"):
        big[name][..., :16] = 0.0
    y, z = quantised(big)
    check_attention(z, *cc.draft_attention4(**y))
    for sign in (13, -13):
        both = dict(x)
        for name, e in (("q", sign), ("k_cache", -sign), ("k_new", -sign)):
            t = x[name].float()
            t[..., :16] *= 2.0 ** e
            t[..., 16:] *= 2.0 ** (0 if dtype == torch.float16 else -e)
            both[name] = t.to(dtype)
        y, z = quantised(both)
        check_attention(z, *cc.draft_attention4(**y))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("power", [-110, 110])
def test_attention4_at_the_ends_of_the_range(cc, dtype, power):
    x = base.inputs(dtype, 2, 9, 4, 2, 64, 500, [500, 129], [tree(9, 2)] * 2, seed=51)
    y, z = quantised(x)
    q = y["q"] * 2.0 ** power
    scale = 0.125 * 2.0 ** -power
    check_attention(z | {"q": q}, *cc.draft_attention4(**(y | {"q": q}), scale=scale), scale=scale)


def test_refused_attention4_structs(cc):
    """What torch tensors never hold, at the C entry point."""
    lib, buf = eng.lib(), torch.zeros(1 << 16, device="cuda")
    at = buf.data_ptr()

    def attention4(**change):
        f = dict(dtype=0, batch=1, q_heads=2, kv_heads=1, head_dim=16, nodes=2, capacity=4, reserved=0, scale=1.0,
                 lens=at, parents=at, lse=at, workspace=at, workspace_bytes=1 << 14)
        f |= {n: base.Rows(at, 64, 64, 16) for n in ("q", "k_new", "v_new", "out")}
        f |= {n: base.Rows(at, 48, 48, 12) for n in ("k_cache", "v_cache")}
        return lib.ckks_draft_attention4(cc.h, ctypes.byref(base.AttentionArgs(**(f | change))), None)

    assert attention4(batch=0) == 0
    for change in (dict(dtype=3), dict(nodes=0), dict(nodes=65), dict(capacity=1 << 30), dict(reserved=1),
                   dict(k_cache=base.Rows(at + 2, 48, 48, 12)), dict(v_cache=base.Rows(at, 48, 48, 14)),
                   dict(v_cache=base.Rows(0, 48, 48, 12)), dict(scale=float("nan")), dict(workspace=at + 4)):
        assert attention4(**change) == 1, change
    assert attention4(capacity=4000, workspace_bytes=16) == 1 and "ckks_draft_attention4_workspace" in lib.ckks_last_error().decode()
    cc.Synchronize()


class Read4Args(ctypes.Structure):
    """ckks_draft_read4_args of include/ckks_b200.h."""
    _fields_ = ([(n, ctypes.c_int32) for n in ("dtype", "batch", "kv_heads", "head_dim", "capacity", "reserved")] +
                [(n, base.Rows) for n in ("cache", "out")] + [("lens", ctypes.c_void_p)])


def test_refused_read4_structs(cc):
    """What torch tensors never hold, at the C entry point."""
    lib, buf = eng.lib(), torch.zeros(1 << 16, device="cuda")
    at = buf.data_ptr()

    def read4(**change):
        f = dict(dtype=0, batch=1, kv_heads=1, head_dim=16, capacity=4, cache=base.Rows(at, 48, 48, 12),
                 out=base.Rows(at + 1024, 64, 64, 16), lens=at + 4096)
        return lib.ckks_draft_read4(cc.h, ctypes.byref(Read4Args(**(f | change))), None)

    assert read4() == 0 and read4(batch=0) == 0 and read4(capacity=0) == 0
    for change in (dict(dtype=3), dict(batch=-1), dict(kv_heads=0), dict(head_dim=257), dict(capacity=-1), dict(lens=0),
                   dict(cache=base.Rows(at + 2, 48, 48, 12)), dict(cache=base.Rows(at, 48, 48, 13)),
                   dict(out=base.Rows(at + 40, 64, 64, 16)), dict(out=base.Rows(0, 64, 64, 16))):
        assert read4(**change) == 1, change
    assert read4(reserved=1) == 1 and "reserved" in lib.ckks_last_error().decode()
    cc.Synchronize()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("n,G", [(1, 4), (7, 3), (13, 4), (40, 2)])
def test_attention4_several_units_a_cta(cc, dtype, D, n, G):
    """Three units and more of unequal lengths for every CTA, of up to 16, 32 and
    64 rows and of two units a head; against the definition in float64 on the
    GPU, as the sizes ask for."""
    Hk, some = 6, [300, 0, 1, 129, 128, 0, 640, 127, 257]
    B = -(-3 * torch.cuda.get_device_properties(0).multi_processor_count // Hk)
    lens = [some[b % len(some)] for b in range(B)]
    parents = tree(n, 2, 1 if n > 1 else 0)
    x = base.inputs(dtype, B, n, G * Hk, Hk, D, 640, lens, [parents] * B, seed=52)
    R = drafting.row4_bytes(D)
    caches = [torch.zeros(B, Hk, 640, R, dtype=torch.uint8, device="cuda") for _ in range(2)]
    for b in range(B):  # every row of the caches, those behind the lengths too
        cc.draft_fill4(*(c[b:b + 1] for c in caches), i32([0]), x["k_cache"][b].transpose(0, 1), x["v_cache"][b].transpose(0, 1),
                       i32([0, 640]))
    y = x | {"k_cache": caches[0], "v_cache": caches[1]}
    out, lse = cc.draft_attention4(**y)
    k, v = (cc.draft_read4(c, i32(lens), D, torch.float32).double() for c in caches)
    see = torch.zeros(n, n, dtype=torch.bool, device="cuda")
    for i, p in enumerate(parents):
        if p >= -1:
            see[i] = see[p] if p >= 0 else False
            see[i, i] = True
    real = see.any(1)
    for b, m in enumerate(lens):
        kk = torch.cat([k[b, :, :m], x["k_new"][b].double().transpose(0, 1)], 1).repeat_interleave(G, 0)
        vv = torch.cat([v[b, :, :m], x["v_new"][b].double().transpose(0, 1)], 1).repeat_interleave(G, 0)
        q = x["q"][b].double().transpose(0, 1)
        hidden = torch.cat([(~real)[:, None].expand(n, m), ~see], 1)
        score = (q @ kk.transpose(1, 2) * D ** -0.5).masked_fill(hidden, -float("inf"))[:, real]
        want_lse = torch.logsumexp(score, 2)
        p = torch.exp(score - want_lse[..., None])
        big = (q.abs() @ kk.abs().transpose(1, 2)).masked_fill(hidden, 0.0)[:, real].amax(2) * D ** -0.5
        keys = (~hidden).sum(1)[real]
        noise = 2.0 ** -23 * ((D + 8) * big + keys + 8)
        room = (2 * HALF[dtype] + noise)[..., None] * (p @ vv.abs()) + 2.0 ** -32 * vv.abs().max() * keys[:, None] + 1e-30
        if dtype == torch.float16:
            room = room + 2.0 ** -25
        off = (out[b].double().transpose(0, 1)[:, real] - p @ vv).abs() / room
        assert (off <= 1.0).all(), f"sequence {b}: {off.max():.3g} times the bound"
        off = (lse[b].double().T[:, real] - want_lse).abs()
        assert (off <= 0.5 * noise + 2.0 ** -22 * (1 + want_lse.abs())).all()
    assert not out[:, ~real].any() and (lse[:, ~real] == -float("inf")).all()
    again = cc.draft_attention4(**y)
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1])
    cc.Synchronize()
