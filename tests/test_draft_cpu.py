"""Argument checks of the drafted-decoding operators, without a GPU: the
Python side before it calls the library, and the C entry points on arguments
that they refuse before any device call."""

import ctypes
from types import SimpleNamespace

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import private_genomic_dnagpt_b200 as eng  # noqa: E402
from private_genomic_dnagpt_b200 import drafting  # noqa: E402

import draft_reference as ref  # noqa: E402


@pytest.fixture
def cc():
    """A context that is not there, on the CPU: good arguments pass the checks
    and are refused by the C entry point."""
    return SimpleNamespace(h=SimpleNamespace(value=0), params=SimpleNamespace(device=-1))


class Reached:
    """A call that passes the checks ends at the null context."""

    def __enter__(self):
        self.inner = pytest.raises(eng.CKKSError, match="null context")
        return self.inner.__enter__()

    def __exit__(self, *e):
        return self.inner.__exit__(*e)


def args(op, t=torch.float32):
    B, n, Hq, Hk, D, cap, V = 2, 3, 4, 2, 8, 10, 6
    q, kn = torch.zeros(B, n, Hq, D, dtype=t), torch.zeros(B, n, Hk, D, dtype=t)
    k = torch.zeros(B, Hk, cap, D, dtype=t)
    lens, parents = torch.zeros(B, dtype=torch.int32), torch.zeros(B, n, dtype=torch.int32)
    p = torch.zeros(B, n + 1, V, dtype=torch.float64)
    return {
        "attention": dict(q=q, k_cache=k, v_cache=k.clone(), lens=lens, k_new=kn, v_new=kn.clone(), parents=parents),
        "verify": dict(target=p, draft=p.float(), tokens=parents, parents=parents,
                       uniforms=torch.zeros(B, n + 1, dtype=torch.float64)),
        "commit": dict(k_cache=k, v_cache=k.clone(), lens=lens, k_new=kn, v_new=kn.clone(), path=parents, count=lens),
        "accumulate": dict(q=q, lse=torch.zeros(B, n, Hq), k_cache=k, lens=lens, path=parents, count=lens,
                           acc=torch.zeros(B, Hk, cap)),
        "evict": dict(k_cache=k, v_cache=k.clone(), acc=torch.zeros(B, Hk, cap), lens=lens, budget=5, recent=2),
    }[op]


OPS = ["attention", "verify", "commit", "accumulate", "evict"]


@pytest.mark.parametrize("op", OPS)
@pytest.mark.parametrize("t", [torch.bfloat16, torch.float16, torch.float32])
def test_good_arguments_reach_the_library(cc, op, t):
    with Reached():
        getattr(drafting, op)(cc, **args(op, t))


@pytest.mark.parametrize("op", OPS)
def test_every_tensor_is_checked(cc, op):
    """Another shape, type, order of the last dimension or a wanted gradient is
    refused, for each tensor in turn."""
    for name, t in args(op).items():
        if not isinstance(t, torch.Tensor):
            continue
        bad = [torch.cat([t, t]), t.to(torch.int64), t[..., None]]
        if t.dim() > 1:
            bad.append(t.expand(2, *t.shape).transpose(0, -1)[..., 0] if t.shape[-1] == 2 else
                       torch.zeros(*t.shape, 2, dtype=t.dtype)[..., 0])
        if t.is_floating_point():
            bad.append(t.clone().requires_grad_())
        for b in bad:
            with pytest.raises(ValueError):
                getattr(drafting, op)(cc, **(args(op) | {name: b}))


@pytest.mark.parametrize("op", OPS)
def test_tensors_of_another_device_are_refused(cc, op):
    cc.params.device = 0
    with pytest.raises(ValueError, match="the context's device"):
        getattr(drafting, op)(cc, **args(op))


def test_written_tensors_have_their_own_memory(cc):
    for op, names in (("commit", ["k_cache", "v_cache"]), ("accumulate", ["acc"])):
        for name in names:
            a = args(op)
            a[name] = a[name][:1].expand_as(a[name])
            with pytest.raises(ValueError, match="share memory"):
                getattr(drafting, op)(cc, **a)
    a = args("evict")
    one = torch.zeros(1, 2, 5, 8).expand(2, 2, 5, 8)
    with pytest.raises(ValueError, match="share memory"):
        drafting.evict(cc, **a, out=(one, one, torch.zeros(2, 2, 5)))


def test_evict_outputs(cc):
    for rows, ok in ((5, True), (9, True), (4, False)):
        out = (torch.zeros(2, 2, rows, 8), torch.zeros(2, 2, rows, 8), torch.zeros(2, 2, rows))
        with Reached() if ok else pytest.raises(ValueError):
            drafting.evict(cc, **args("evict"), out=out)


def test_c_entry_points_refuse_null():
    lib = eng.lib()
    for name in ("attention", "verify", "commit", "accumulate", "evict"):
        assert getattr(lib, "ckks_draft_" + name)(None, ctypes.create_string_buffer(512), None) == 1
        assert b"null context" in lib.ckks_last_error()
    for name in ("attention", "evict"):
        assert getattr(lib, f"ckks_draft_{name}_workspace")(None, ctypes.create_string_buffer(512)) == -1
    assert lib.ckks_block_set_drafts(None, None, 0, 0) == 1


def test_reference_is_self_consistent():
    """The float64 definitions on cases known by hand."""
    assert ref.ancestors([-1, 0, 1, 5, -2, 4], 2) == [0, 1, 2]
    assert ref.ancestors([-1, 0, 1, 5, -2, 4], 5) == [] and ref.ancestors([-1, 0, 1, 5, -2, 4], 3) == []
    assert list(ref.keep(np.array([3.0, 1.0, 3.0, 2.0, 0.0]), 5, 3, 1)) == [0, 2, 4]
    p, q = np.array([[[0.0, 1.0], [0.5, 0.5]]]), np.array([[[1.0, 0.0], [0.5, 0.5]]])
    path, count, token = ref.verify(p, q, np.array([[0]]), np.array([[-1]]), np.array([[0.1, 0.3]]))
    assert count[0] == 0 and token[0] == 1 and ctypes.sizeof(ctypes.c_int32) == 4
