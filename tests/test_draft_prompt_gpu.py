"""Causal attention within packed prompts, and their rows appended to a cache,
on the GPU against their definitions in float64 (tests/prompt_reference.py).

Bounds as for the attention of a tree (tests/test_draft_gpu.py): the weights
may be rounded to the tensors' type (half a step u), the result is (u), scores
carry D + 8 roundings of 2^-24 on sum |q k| scale and a sum over N keys N + 8
more, each at most doubled by the division."""

import ctypes

import numpy as np
import pytest

import prompt_reference as ref

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import private_genomic_dnagpt_b200 as eng  # noqa: E402

from test_draft_gpu import HALF, TYPES, f64, i32  # noqa: E402


@pytest.fixture(scope="module")
def cc():
    return eng.GenCryptoContext(eng.CCParams(ring_dim_log=10, limbs=3, dnum=1, seed=3))


def packed(lengths, first=0):
    return [first] + [first + int(x) for x in np.cumsum(lengths)]


def inputs(dtype, T, Hq, Hk, D, starts, seed=0, spread=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *s: (spread * torch.randn(*s, generator=g, device="cuda")).to(dtype)  # noqa: E731
    return dict(q=normal(T, Hq, D), k=normal(T, Hk, D), v=normal(T, Hk, D), starts=i32(starts))


def check(x, out, lse, scale=None):
    q = f64(x["q"])
    D = q.shape[2]
    scale = D ** -0.5 if scale is None else scale
    want, wlse, mag, big, keys = ref.prompt(q, f64(x["k"]), f64(x["v"]), x["starts"].cpu().numpy(), scale)
    got, glse = f64(out), f64(lse)
    noise = 2.0 ** -23 * ((D + 8) * big + keys + 8)
    room = (2 * HALF[x["q"].dtype] + noise)[..., None] * mag + 1e-30
    assert np.isfinite(got).all()
    worst = (np.abs(got - want) / room).max() if got.size else 0.0
    assert worst <= 1.0, f"out: {worst:.3g} times the bound"
    seen = keys > 0
    assert np.array_equal(glse == -np.inf, ~seen) and not got[~seen].any()
    assert (np.abs(glse[seen] - wlse[seen]) <= (0.5 * noise + 2.0 ** -22 * (1 + np.abs(wlse)))[seen]).all()


SHAPES = [
    # lengths, first row, rows behind the last, Hq, Hk, D
    ([103], 0, 0, 12, 12, 64),
    ([1], 0, 0, 1, 1, 64),
    ([1, 0, 2, 1], 0, 0, 2, 1, 64),
    ([0, 0], 0, 5, 2, 2, 64),                  # no sequence has rows
    ([127, 128, 129], 3, 7, 4, 2, 64),
    ([255, 256, 257, 1, 64, 65, 63], 0, 1, 4, 1, 128),
    ([640], 0, 0, 8, 8, 128),
    ([1000, 513, 0, 385], 0, 40, 6, 3, 64),
    ([1537], 0, 0, 4, 1, 128),
    ([300, 20], 0, 0, 2, 1, 256),
    ([200, 333], 1, 0, 3, 3, 192),
    ([130], 0, 0, 4, 2, 80),
    ([390, 7], 0, 0, 2, 2, 96),
    ([140], 0, 0, 2, 2, 32),
    ([260, 31], 0, 2, 2, 1, 8),
    ([100, 70], 0, 0, 2, 1, 5),                # odd head sizes
    ([66], 0, 0, 5, 5, 33),
    ([190, 64], 0, 0, 2, 2, 100),
    ([65], 0, 0, 2, 1, 1),
    ([530], 0, 0, 2, 2, 248),
    ([300], 0, 0, 3, 1, 136),
    ([(37 * i) % 201 for i in range(70)], 0, 0, 2, 2, 64),   # many sequences
    ([1] * 100, 0, 0, 3, 3, 128),
    ([2, 900] * 20, 5, 5, 1, 1, 64),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(map(str, [len(s[0]), sum(s[0]), *s[1:]])))
def test_prompt(cc, dtype, shape):
    lengths, first, spare, Hq, Hk, D = shape
    starts = packed(lengths, first)
    x = inputs(dtype, starts[-1] + spare, Hq, Hk, D, starts)
    check(x, *cc.draft_prompt(**x))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 128])
def test_long_prompt(cc, dtype, D):
    starts = packed([4100, 2049])
    x = inputs(dtype, starts[-1], 2, 1, D, starts, seed=1)
    check(x, *cc.draft_prompt(**x))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 128, 200])
def test_sharp_rows_and_scales(cc, dtype, D):
    """Scores far apart: the running maximum moves by hundreds."""
    starts = packed([700, 333])
    x = inputs(dtype, starts[-1], 4, 2, D, starts, seed=2, spread=6.0)
    check(x, *cc.draft_prompt(**x))
    for scale in (0.5, -0.01, 0.0):
        check(x, *cc.draft_prompt(**x, scale=scale), scale=scale)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("scale", [0.0, 2.0 ** -112])
def test_scales_that_undo_large_scores(cc, dtype, scale):
    """Scores around 2^115: with a scale of 0 every key weighs the same."""
    starts = packed([200, 70])
    x = inputs(dtype, starts[-1], 4, 2, 64, starts, seed=3)
    x["q"] = x["q"] * 2.0 ** 56
    x["k"] = x["k"] * 2.0 ** 56
    check(x, *cc.draft_prompt(**x, scale=scale), scale=scale)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rising", [True, False])
def test_rows_of_rising_scores(cc, dtype, rising):
    """Each key's score is above (below) the one before it by 3 / 2, so the
    reference point moves in every tile."""
    n, D = 900, 64
    x = inputs(dtype, n, 1, 1, D, [0, n], seed=3)
    x["q"].zero_()
    x["k"].zero_()
    x["q"][..., 0] = 1.0
    steps = 1.5 * (torch.arange(n, device="cuda", dtype=torch.float32) - (n if rising else 0))
    # two parts, so that 16-bit keys hold the whole step
    hi = torch.floor(steps / 16) * 16
    x["q"][..., 1] = 1.0
    x["k"][:, 0, 0], x["k"][:, 0, 1] = hi.to(dtype), (steps - hi).to(dtype)
    if not rising:
        x["k"] = -x["k"]
    check(x, *cc.draft_prompt(**x, scale=1.0), scale=1.0)


@pytest.mark.parametrize("dtype", TYPES)
def test_starts_out_of_order(cc, dtype):
    """A start below an earlier one, below 0 or past the rows is taken as the
    nearest that keeps the order."""
    for starts in ([0, 100, 50, 120], [-7, 40, 1000], [90, 10, 300], [500, 600], [-2 ** 31, 2 ** 31 - 1]):
        x = inputs(dtype, 260, 2, 1, 64, starts, seed=4)
        check(x, *cc.draft_prompt(**x))


@pytest.mark.parametrize("dtype", TYPES)
def test_nothing_to_do(cc, dtype):
    x = inputs(dtype, 10, 2, 1, 64, [0])
    out, lse = cc.draft_prompt(**x)  # no sequence
    assert not out.any() and (lse == -float("inf")).all()
    x = inputs(dtype, 0, 2, 1, 64, [0, 0])
    out, lse = cc.draft_prompt(**x)
    assert out.shape == (0, 2, 64) and lse.shape == (0, 2)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [33, 64, 128, 200])
@pytest.mark.parametrize("at", [0, 5, 127, 128, 130, 255, 300, 399])
def test_what_a_row_does_not_see_does_not_reach_it(cc, dtype, D, at):
    """A row whose key and value are NaN, and whose values are infinite, shows
    in itself and the rows behind it, whatever its weight, and in no other."""
    starts = packed([400, 200], 1)
    x = inputs(dtype, starts[-1] + 2, 4, 2, D, starts, seed=5)
    for name in ("q", "k"):
        x[name][..., 0] = 0.0
    x["q"][..., 0] = D ** 0.5
    clean, clse = cc.draft_prompt(**x)
    for value in (float("nan"), float("inf")):
        y = {k: v.clone() for k, v in x.items()}
        y["v"][1 + at, :, 0] = value
        y["k"][1 + at, :, 0] = -1000.0
        out, lse = cc.draft_prompt(**y)
        bad = slice(1 + at, 401)
        assert not torch.isfinite(out[bad][..., 0]).any()
        assert torch.isfinite(out[bad][..., 1:]).all() and torch.isfinite(lse[bad]).all()
        same = torch.ones(len(out), dtype=torch.bool, device="cuda")
        same[bad] = False
        assert torch.equal(out[same], clean[same]) and torch.equal(lse[same], clse[same])
    y = {k: v.clone() for k, v in x.items()}
    y["k"][1 + at] = float("nan")
    out, lse = cc.draft_prompt(**y)
    assert torch.isnan(out[bad]).all() and torch.isnan(lse[bad]).all()
    assert torch.equal(out[same], clean[same]) and torch.equal(lse[same], clse[same])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 128, 40])
def test_rows_of_no_sequence_are_not_read(cc, dtype, D):
    starts = packed([130, 257], 9)
    x = inputs(dtype, starts[-1] + 200, 2, 2, D, starts, seed=6)
    clean = cc.draft_prompt(**x)
    for name in ("q", "k", "v"):
        x[name][:9] = float("nan")
        x[name][starts[-1]:] = float("inf")
    got = cc.draft_prompt(**x)
    assert torch.equal(clean[0], got[0]) and torch.equal(clean[1], got[1])


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_alignment(cc, dtype):
    starts = packed([210, 111])
    x = inputs(dtype, 321, 4, 2, 64, starts, seed=7)
    want = cc.draft_prompt(**x)
    y = dict(x)
    y["q"] = x["q"].transpose(0, 1).contiguous().transpose(0, 1)
    both = torch.cat([x["k"], x["v"]], 1)  # one buffer for keys and values
    y["k"], y["v"] = both[:, :2], both[:, 2:]
    got = cc.draft_prompt(**y)
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
    wide = torch.zeros(321, 2, 72, dtype=dtype, device="cuda")
    wide[..., :64] = x["v"]
    got = cc.draft_prompt(**(dict(x) | {"v": wide[..., :64]}))
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
    for name in ("q", "k", "v"):  # one element off every wide boundary
        flat = torch.zeros(x[name].numel() + 1, dtype=dtype, device="cuda")
        flat[1:] = x[name].reshape(-1)
        z = dict(x) | {name: flat[1:].view(x[name].shape)}
        check(z, *cc.draft_prompt(**z))
    one = dict(x) | {"k": x["k"][:, :1].expand(321, 2, 64)}  # one head for both
    check(one, *cc.draft_prompt(**one))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_offsets_past_32_bits(cc, dtype):
    """Rows 2^25 elements apart: the last ones lie past 2^31 elements."""
    step, T = 1 << 25, 70
    store = torch.empty(step * T, dtype=dtype, device="cuda")
    x = inputs(dtype, T, 2, 2, 64, [0, 66, 70], seed=8)
    for i, name in enumerate(("q", "k", "v")):
        view = torch.as_strided(store, (T, 2, 64), (step, 64, 1), 4096 * i)
        view.copy_(x[name])
        x[name] = view
    check(x, *cc.draft_prompt(**x))


@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 64), (torch.float16, 128), (torch.float32, 64), (torch.bfloat16, 33)])
def test_repeats_streams_and_graphs(cc, dtype, D):
    """The same bits again, on another stream, and from two captured calls
    replayed side by side with new starts."""
    starts = [packed([1000, 300, 0, 700]), packed([600, 1100, 200, 50])]
    xs = [inputs(dtype, 2000, 4, 2, D, s, seed=9 + i) for i, s in enumerate(starts)]
    want = [cc.draft_prompt(**x) for x in xs]
    again = cc.draft_prompt(**xs[0])
    assert torch.equal(again[0], want[0][0]) and torch.equal(again[1], want[0][1])
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = cc.draft_prompt(**xs[0])
    s.synchronize()
    assert torch.equal(got[0], want[0][0])
    graphs, outs = [], []
    for x in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(cc.draft_prompt(**x))
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
    xs[0]["starts"].copy_(i32(starts[1]))  # the lengths are the device's
    graphs[0].replay()
    torch.cuda.synchronize()
    check(xs[0], *outs[0])


def test_matches_the_tree_of_a_chain(cc):
    """A prompt is a chain of nodes over an empty cache."""
    for dtype in TYPES:
        x = inputs(dtype, 64, 4, 2, 64, [0, 64], seed=12)
        out, lse = cc.draft_prompt(**x)
        empty = torch.zeros(1, 2, 0, 64, dtype=dtype, device="cuda")
        chain = torch.arange(-1, 63, dtype=torch.int32, device="cuda")[None]
        want, wlse = cc.draft_attention(x["q"][None], empty, empty, i32([0]), x["k"][None], x["v"][None], chain)
        assert (out.double() - want[0].double()).abs().max() <= 4 * HALF[dtype] * want.abs().max() + 1e-5
        assert (lse - wlse[0]).abs().max() <= 1e-5


# ---- fill -----------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 80, 33, 1])
def test_fill(cc, dtype, D):
    """Ragged sequences behind what is cached; those that do not fit are left
    as they are and reported."""
    lengths, lens, cap = [17, 0, 1, 40, 16, 33], [3, 5, 0, 24, 48, 32], 64
    starts = packed(lengths, 2)
    x = inputs(dtype, starts[-1] + 3, 2, 2, D, starts, seed=13)
    g = torch.Generator(device="cuda").manual_seed(14)
    cache = [torch.randn(6, 2, cap, D, generator=g, device="cuda").to(dtype) for _ in range(2)]
    want = [ref.fill(f64(c), lens, f64(x[n]), starts) for c, n in zip(cache, ("k", "v"))]
    got = cc.draft_fill(*cache, i32(lens), x["k"], x["v"], x["starts"])
    assert np.array_equal(got.cpu().numpy(), want[0][1]) and got.tolist() == [20, 5, 1, 64, 64, 32]
    for c, w in zip(cache, want):
        assert np.array_equal(f64(c), w[0])
    with pytest.raises(eng.CKKSError, match=r"1 sequence\(s\) left unchanged"):
        cc.Synchronize()
    cc.Synchronize()


def test_fill_odd_lengths_and_starts(cc):
    k = torch.ones(50, 1, 8, device="cuda")
    cache = torch.zeros(4, 1, 20, 8, device="cuda"), torch.zeros(4, 1, 20, 8, device="cuda")
    lens = cc.draft_fill(*cache, i32([-1, 21, 0, 0]), k, 2 * k, i32([0, 5, 10, 7, 99]))
    # the last sequence has 40 rows, from 10 to the end; the third has none
    assert lens.tolist() == [-1, 21, 0, 0] and not cache[0].any()
    with pytest.raises(eng.CKKSError, match=r"3 sequence\(s\)"):
        cc.Synchronize()
    assert cc.draft_fill(*cache, i32([0] * 4), k, k, i32([0] * 5)).tolist() == [0] * 4
    assert cc.draft_fill(cache[0][:0], cache[1][:0], i32([]), k, k, i32([0])).shape == (0,)
    none = torch.zeros(4, 1, 0, 8, device="cuda")
    assert cc.draft_fill(none, none.clone(), i32([0] * 4), k[:0], k[:0], i32([0] * 5)).tolist() == [0] * 4
    cc.Synchronize()


def test_fill_of_many_sequences(cc):
    B = 100
    lengths = [(7 * i) % 40 for i in range(B)]
    starts = packed(lengths)
    x = inputs(torch.bfloat16, starts[-1], 3, 3, 64, starts, seed=15)
    cache = [torch.zeros(B, 3, 48, 64, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    lens = [i % 9 for i in range(B)]
    want = [ref.fill(f64(c), lens, f64(x[n]), starts) for c, n in zip(cache, ("k", "v"))]
    got = cc.draft_fill(*cache, i32(lens), x["k"], x["v"], x["starts"])
    assert np.array_equal(got.cpu().numpy(), want[0][1])
    for c, w in zip(cache, want):
        assert np.array_equal(f64(c), w[0])
    cc.Synchronize()


class Rows(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p)] + [(n, ctypes.c_int64) for n in ("batch", "head", "row")]


class PromptArgs(ctypes.Structure):
    """ckks_draft_prompt_args of include/ckks_b200.h."""
    _fields_ = ([(n, ctypes.c_int32) for n in ("dtype", "batch", "q_heads", "kv_heads", "head_dim", "tokens")] +
                [("scale", ctypes.c_double)] + [(n, Rows) for n in ("q", "k", "v", "out")] +
                [("starts", ctypes.c_void_p), ("lse", ctypes.c_void_p)])


def test_prompt_c_entry_point(cc):
    """The C struct, an output in another order of dimensions, the refusals."""
    x = inputs(torch.bfloat16, 150, 4, 2, 64, [0, 100, 149], seed=16)
    want, wlse = cc.draft_prompt(**x)
    out, lse = torch.zeros(4, 150, 64, dtype=torch.bfloat16, device="cuda"), torch.zeros(150, 4, device="cuda")
    rows = lambda t: Rows(t.data_ptr(), 0, t.stride(1), t.stride(0))  # noqa: E731
    good = dict(dtype=0, batch=2, q_heads=4, kv_heads=2, head_dim=64, tokens=150, scale=0.125, q=rows(x["q"]),
                k=rows(x["k"]), v=rows(x["v"]), out=rows(out.transpose(0, 1)), starts=x["starts"].data_ptr(),
                lse=lse.data_ptr())
    call = lambda **more: eng.lib().ckks_draft_prompt(cc.h, ctypes.byref(PromptArgs(**(good | more))), None)  # noqa: E731
    torch.cuda.synchronize()
    assert call() == 0
    torch.cuda.synchronize()
    assert torch.equal(out.transpose(0, 1), want) and torch.equal(lse, wlse)
    for more in (dict(dtype=3), dict(batch=-1), dict(q_heads=3), dict(kv_heads=0), dict(head_dim=0), dict(head_dim=257),
                 dict(tokens=-1), dict(scale=float("nan")), dict(scale=float("inf")), dict(starts=None), dict(lse=None),
                 dict(q=Rows(0, 0, 64, 256)), dict(k=Rows(x["k"].data_ptr() + 1, 0, 64, 128)),
                 dict(v=Rows(x["v"].data_ptr(), 0, -64, 128)), dict(tokens=(1 << 30) - 1, q_heads=4096)):
        assert call(**more) == 1, more
    assert call(tokens=0) == 0
    cc.Synchronize()


@pytest.mark.parametrize("D", [64, 128, 40])
def test_a_weight_of_nothing_is_nothing(cc, D):
    """Keys whose scores lie 1000 below the others' have the weight 0 in 32 bits,
    so that the largest values of bfloat16 do not show through them."""
    starts = packed([500, 300])
    x = inputs(torch.bfloat16, starts[-1], 2, 1, D, starts, seed=20)
    for name in ("q", "k"):
        x[name][..., 0] = 0.0
    x["q"][..., 0] = D ** 0.5
    for first in (0, 500):
        x["k"][first + 1:first + 70, :, 0] = -1000.0
        x["v"][first + 1:first + 70] = 3e38
    check(x, *cc.draft_prompt(**x))
    x["k"][first + 1:first + 70, :, 0] = -3e38  # scores of -inf
    y = dict(x) | {"v": x["v"].clone()}
    y["v"][first + 1:first + 70] = 0.0
    got, want = cc.draft_prompt(**x), cc.draft_prompt(**y)
    assert torch.equal(got[0][500:], want[0][500:]) and torch.equal(got[1][500:], want[1][500:])


def sms():
    return torch.cuda.get_device_properties(0).multi_processor_count


def check_exactly(x, out, lse, scale):
    """``check`` with the definition in float64 on the GPU, as the sizes ask
    for; elements that see a value that is no number are none."""
    q, k, v = (x[n].double() for n in ("q", "k", "v"))
    T, Hq, D = q.shape
    G = Hq // k.shape[1]
    k, v = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    bad = ~torch.isfinite(v)
    v = torch.where(bad, 0.0, v)
    s = ref.starts_of(x["starts"].cpu().numpy(), T)
    seen = torch.zeros(T, dtype=torch.bool, device="cuda")
    for a, e in zip(s, s[1:]):
        if a == e:
            continue
        seen[a:e] = True
        n = e - a
        above = torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1)
        for h in range(0, Hq, 8):
            qq, kk, vv = (t[a:e, h:h + 8].transpose(0, 1) for t in (q, k, v))
            score = (qq @ kk.transpose(1, 2) * scale).masked_fill(above, -float("inf"))
            want_lse = torch.logsumexp(score, 2)
            p = torch.exp(score - want_lse[..., None])
            big = (qq.abs() @ kk.abs().transpose(1, 2)).masked_fill(above, 0.0).amax(2) * abs(scale)
            noise = 2.0 ** -23 * ((D + 8) * big + torch.arange(1, n + 1, device="cuda") + 8)
            room = (2 * HALF[x["q"].dtype] + noise)[..., None] * (p @ vv.abs()) + 1e-30
            got = out[a:e, h:h + 8].transpose(0, 1).double()
            none = bad[a:e, h:h + 8].transpose(0, 1).cumsum(1) > 0
            assert not torch.isfinite(got[none]).any()
            off = torch.where(none, 0.0, (got - p @ vv).abs() / room)  # (a NaN fails too)
            assert (off <= 1.0).all(), f"rows {a} to {e}, heads from {h}: {off.max():.3g} times the bound"
            off = (lse[a:e, h:h + 8].T.double() - want_lse).abs()
            assert (off <= 0.5 * noise + 2.0 ** -22 * (1 + want_lse.abs())).all()
    assert not out[~seen].any() and (lse[~seen] == -float("inf")).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128, 192, 256])
@pytest.mark.parametrize("spoiled", [False, True])
def test_several_units_a_cta(cc, dtype, D, spoiled):
    """Three units and more of unequal lengths for every CTA of the tensor-core
    kernel, with both row groups and one; then with values that are no numbers next
    to the causal border in some of the units."""
    lengths, rows = [1, 120, 129, 257, 0, 700, 1500], 256 if D <= 128 else 128
    units = sum(-(-n // rows) for n in lengths)
    Hk = 4
    Hq = Hk * -(-3 * sms() // (units * Hk))
    assert units * Hq >= 3 * sms()
    starts = packed(lengths, 2)
    x = inputs(dtype, starts[-1] + 3, Hq, Hk, D, starts, seed=21)
    if spoiled:
        for seq, at, head, d in ((2, 100, 0, 3), (2, 128, 3, 5), (3, 127, 1, 1), (3, 200, 1, D - 1), (3, 256, 0, 9),
                                 (5, 130, 2, 0), (5, 255, 1, 7), (5, 256, 3, 11), (5, 699, 0, 2), (6, 600, 3, 4),
                                 (6, 1279, 1, 6), (6, 1280, 2, 8), (6, 1407, 0, 13), (6, 1499, 1, 15)):
            x["v"][starts[seq] + at, head, d] = float("nan") if at % 2 else float("inf")
    out, lse = cc.draft_prompt(**x)
    check_exactly(x, out, lse, D ** -0.5)
    again = cc.draft_prompt(**x)
    fine = torch.isfinite(out)
    assert torch.equal(fine, torch.isfinite(again[0])) and torch.equal(out[fine], again[0][fine]) and torch.equal(lse, again[1])
    cc.Synchronize()


@pytest.mark.parametrize("dtype,D", [(torch.float32, 128), (torch.float32, 100), (torch.float32, 65), (torch.bfloat16, 100),
                                     (torch.float16, 128)])
@pytest.mark.parametrize("scale", [None, -0.05])
def test_tall_tiles_on_the_cuda_cores(cc, dtype, D, scale):
    """Heads of 65 to 128 in as many rows and heads as the kernel takes 128 rows
    at a time for; in 16 bits off every wide boundary."""
    lengths = [1, 63, 64, 65, 127, 128, 129, 500]
    starts = packed(lengths, 1)
    T = starts[-1] + 2
    Hk = 8
    Hq = Hk * -(-(3 * sms() // 2) // (T // 128 * Hk))
    assert T // 128 * Hq >= 3 * sms() // 2
    x = inputs(dtype, T, Hq, Hk, D, starts, seed=22)
    if dtype != torch.float32:
        flat = torch.zeros(x["k"].numel() + 1, dtype=dtype, device="cuda")
        flat[1:] = x["k"].reshape(-1)
        x["k"] = flat[1:].view(x["k"].shape)
    out, lse = cc.draft_prompt(**x, scale=scale)
    check_exactly(x, out, lse, D ** -0.5 if scale is None else scale)
    # what only the last rows of two sequences see, and rows of no sequence
    y = {k: v.clone() if dtype == torch.float32 else v for k, v in x.items()}
    for at in (starts[5] + 120, starts[8] - 3):
        for name in ("k", "v"):
            y[name][at] = float("nan")
    y["q"][0] = y["k"][0] = y["v"][0] = y["v"][T - 1] = float("nan")
    got, glse = cc.draft_prompt(**y, scale=scale)
    bad = torch.zeros(T, dtype=torch.bool, device="cuda")
    bad[starts[5] + 120:starts[6]] = bad[starts[8] - 3:starts[8]] = True
    assert torch.isnan(got[bad]).all() and torch.isnan(glse[bad]).all()
    assert torch.equal(got[~bad], out[~bad]) and torch.equal(glse[~bad], lse[~bad])
    cc.Synchronize()


@pytest.mark.parametrize("dtype", TYPES)
def test_prompts_and_fills_from_two_threads(cc, dtype):
    """Calls of other sizes at the same time from two host threads."""
    import threading
    runs, wrong = [], []
    for lengths, H, D in (([700, 129], 4, 64), ([90, 300], 2, 200)):
        starts = packed(lengths)
        x = inputs(dtype, starts[-1], H, H, D, starts, seed=23)
        zero, st = i32([0, 0]), x["starts"]

        def call(x=x, H=H, D=D, zero=zero, st=st):
            caches = [torch.zeros(2, H, 700, D, dtype=dtype, device="cuda") for _ in range(2)]
            return (*cc.draft_prompt(**x), cc.draft_fill(*caches, zero, x["k"], x["v"], st), *caches)

        runs.append((call, call()))
    torch.cuda.synchronize()

    def calls(call, want):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(50):
                got = call()
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want)):
                    wrong.append(1)

    threads = [threading.Thread(target=calls, args=r) for r in runs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
    cc.Synchronize()
