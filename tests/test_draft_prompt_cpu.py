"""Argument checks of packed prompts and 4-bit caches, without a GPU, and the
definitions of tests/prompt_reference.py on cases known by hand."""

import ctypes

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import private_genomic_dnagpt_b200 as eng  # noqa: E402
from private_genomic_dnagpt_b200 import drafting  # noqa: E402

import prompt_reference as ref  # noqa: E402
from test_draft_cpu import Reached, cc  # noqa: E402, F401

OPS = ["prompt", "fill", "fill4", "commit4", "read4", "attention4"]


def args(op, t=torch.float32):
    B, n, T, Hq, Hk, D, cap = 2, 3, 7, 4, 2, 8, 10
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    four = torch.zeros(B, Hk, cap, 12, dtype=torch.uint8)
    k = torch.zeros(T, Hk, D, dtype=t)
    kn = torch.zeros(B, n, Hk, D, dtype=t)
    plain = torch.zeros(B, Hk, cap, D, dtype=t)
    return {
        "prompt": dict(q=torch.zeros(T, Hq, D, dtype=t), k=k, v=k.clone(), starts=i32(B + 1)),
        "fill": dict(k_cache=plain, v_cache=plain.clone(), lens=i32(B), k=k, v=k.clone(), starts=i32(B + 1)),
        "fill4": dict(k_cache=four, v_cache=four.clone(), lens=i32(B), k=k, v=k.clone(), starts=i32(B + 1)),
        "commit4": dict(k_cache=four, v_cache=four.clone(), lens=i32(B), k_new=kn, v_new=kn.clone(), path=i32(B, n),
                        count=i32(B)),
        "read4": dict(cache=four, lens=i32(B), head_dim=D, dtype=t),
        "attention4": dict(q=torch.zeros(B, n, Hq, D, dtype=t), k_cache=four, v_cache=four.clone(), lens=i32(B), k_new=kn,
                           v_new=kn.clone(), parents=i32(B, n)),
    }[op]


@pytest.mark.parametrize("op", OPS)
@pytest.mark.parametrize("t", [torch.bfloat16, torch.float16, torch.float32])
def test_good_arguments_reach_the_library(cc, op, t):  # noqa: F811
    with Reached():
        getattr(drafting, op)(cc, **args(op, t))


@pytest.mark.parametrize("op", OPS)
def test_every_tensor_is_checked(cc, op):  # noqa: F811
    """Another shape, type, order of the last dimension or a wanted gradient of
    either mode, and a negated view, are refused for each tensor in turn."""
    import torch.autograd.forward_ad as fwd
    for name, t in args(op).items():
        if not isinstance(t, torch.Tensor):
            continue
        bad = [t.to(torch.int64), t[..., None], t[..., :0]]
        if not (op == "prompt" and name == "starts"):  # any number of sequences
            bad.append(torch.cat([t, t]))
        if t.dim() > 1:
            bad.append(torch.zeros(*t.shape, 2, dtype=t.dtype)[..., 0])
        if t.is_floating_point():
            bad += [t.clone().requires_grad_(), torch._neg_view(t), t.double()]
        for b in bad:
            with pytest.raises(ValueError):
                getattr(drafting, op)(cc, **(args(op) | {name: b}))
        if t.is_floating_point():
            with fwd.dual_level(), torch.no_grad(), pytest.raises(ValueError, match="forward-mode"):
                getattr(drafting, op)(cc, **(args(op) | {name: fwd.make_dual(t, torch.ones_like(t))}))


@pytest.mark.parametrize("op", OPS)
def test_tensors_of_another_device_are_refused(cc, op):  # noqa: F811
    cc.params.device = 0
    with pytest.raises(ValueError, match="the context's device"):
        getattr(drafting, op)(cc, **args(op))


@pytest.mark.parametrize("op", ["fill", "fill4", "commit4"])
@pytest.mark.parametrize("name", ["k_cache", "v_cache"])
def test_written_tensors_have_their_own_memory(cc, op, name):  # noqa: F811
    a = args(op)
    a[name] = a[name][:1].expand_as(a[name])
    with pytest.raises(ValueError, match="share memory"):
        getattr(drafting, op)(cc, **a)


def test_head_sizes_and_types_of_4_bit_rows(cc):  # noqa: F811
    for D in (1, 16, 17, 64, 80, 128, 256):
        assert drafting.row4_bytes(D) == ref.row_bytes(D)
    for D in (0, -1, 257, 1 << 40):
        with pytest.raises(ValueError, match="head_dim outside"):
            drafting.row4_bytes(D)
        with pytest.raises(ValueError):
            drafting.read4(cc, **(args("read4") | {"head_dim": D}))
    for t in (torch.float64, torch.uint8, torch.int32):
        with pytest.raises(ValueError, match="expected bfloat16, float16 or float32"):
            drafting.read4(cc, **(args("read4") | {"dtype": t}))
    with pytest.raises(ValueError):
        drafting.read4(cc, **(args("read4") | {"head_dim": 17}))


def test_sizes_past_32_bits(cc):  # noqa: F811
    a = args("attention4")
    for name in ("k_cache", "v_cache"):
        a[name] = a[name][:, :, :1].expand(2, 2, 2 ** 32 + 10, 12)
    with pytest.raises(ValueError, match="capacity: 4294967306"):
        drafting.attention4(cc, **a)
    a = args("prompt")
    for name in ("q", "k", "v"):
        a[name] = a[name][:1].expand(2 ** 32 + 7, *a[name].shape[1:])
    with pytest.raises((ValueError, RuntimeError)):
        drafting.prompt(cc, **a)


def test_c_entry_points_refuse_null():
    lib = eng.lib()
    for name in ("prompt", "fill", "fill4", "commit4", "read4", "attention4"):
        assert getattr(lib, "ckks_draft_" + name)(None, ctypes.create_string_buffer(512), None) == 1
        assert b"null context" in lib.ckks_last_error()
    assert lib.ckks_draft_attention4_workspace(None, ctypes.create_string_buffer(512)) == -1
    assert lib.ckks_draft_row4_bytes(64) == 36 and lib.ckks_draft_row4_bytes(0) == -1


def test_reference_on_cases_known_by_hand():
    assert ref.SCALES[8] == 2.0 ** -14 and ref.SCALES[-1] == 10240 and ref.SCALES[1] == 2.0 ** -17
    x = np.zeros((1, 16))
    x[0, :9] = [6.0, 5.0, 2.5, 1.75, 1.25, 0.75, 0.25, -3.5, -0.2]
    row = ref.pack(x)
    assert row.shape == (1, 12) and row[0, 8] == 15 * 8  # a scale of 1
    assert ref.unpack(row, 16)[0, :9].tolist() == [6.0, 4.0, 2.0, 2.0, 1.0, 1.0, 0.0, -4.0, -0.0]
    assert row[0, 0] == 7 + 16 * 6 and row[0, 4] == 8  # 6 and 4; -0 and 0
    out, lse, *_ = ref.prompt(np.ones((3, 1, 1)), np.zeros((3, 1, 1)), np.array([1.0, 3.0, 9.0]).reshape(3, 1, 1),
                              [0, 2, 1], 1.0)
    assert out[:, 0, 0].tolist() == [1.0, 2.0, 0.0] and lse[2, 0] == -np.inf and abs(lse[1, 0] - np.log(2)) < 1e-15
