"""Drafted decoding on the data owner's side.

An encrypted forward costs about the same for one token as for the 32 tokens
that share a ciphertext, so the data owner drafts several tokens with a small
plain model, has the encrypted model evaluate all of them in one forward and
keeps those that its probabilities confirm.  The operators between two
forwards run on the owner's GPU, on torch tensors of the context's device and
on torch's current stream (``CryptoContext`` offers them as methods):

  draft_attention    a tree of drafted nodes over the draft model's cache
  draft_verify       which drafts the target confirms, and the next token
  draft_commit       the accepted rows appended to the cache
  draft_accumulate   the attention weight they give each cached key
  draft_evict        the cache cut to its latest and heaviest keys

``DraftModel`` is the plain draft model: blocks of the same weights that
``EncryptedBlock`` takes, evaluated with these operators; it stands beside
``EncryptedModel``, whose ``forward(x, parents)`` evaluates the drafts.

Trees: ``parents[b, i]`` is -1 (the node follows the cached tokens directly)
or an earlier node; a node with any other parent is padding.  None of the
operators has a gradient, allocates outside torch or waits for the GPU, and
each can be captured into a CUDA graph.
"""

from __future__ import annotations

import math
import struct

MAX_NODES = 64  # nodes of one tree

_DTYPES: dict = {}
_ATTENTION = struct.Struct("8id24q5q")
_VERIFY = struct.Struct("6i8q6q")
_COMMIT = struct.Struct("6i16q4q")
_ACCUMULATE = struct.Struct("8id12q4q")
_EVICT = struct.Struct("8i24q5q")


def _torch():
    import torch
    if not _DTYPES:
        _DTYPES.update({torch.bfloat16: 0, torch.float16: 1, torch.float32: 2, torch.float64: 3})
    return torch


def _refuse(name, why):
    raise ValueError(f"{name}: {why}")


def _tensor(t, name, shape, dtype, device, contiguous=False):
    """Checks one argument and returns it."""
    if t.shape != shape:
        _refuse(name, f"expected the shape {tuple(shape)}, got {tuple(t.shape)}")
    if t.dtype is not dtype:
        _refuse(name, f"expected {dtype}, got {t.dtype}")
    if t.device != device:
        _refuse(name, f"expected a tensor of {device}, the context's device, got {t.device}")
    if t.requires_grad and _torch().is_grad_enabled():
        _refuse(name, "requires a gradient, which this operator does not have (call it under torch.no_grad)")
    if contiguous and not t.is_contiguous():
        _refuse(name, "must be contiguous")
    if t.shape and t.shape[-1] > 1 and t.stride(-1) != 1 and t.numel():
        _refuse(name, "its last dimension must be contiguous")
    return t


def _writable(t, name):
    """Refuses a tensor of which two elements share memory."""
    for n, s in zip(t.shape, t.stride()):
        if n > 1 and s == 0:
            _refuse(name, "is written, but some of its elements share memory")
    return t


def _device(cc):
    d = cc._draft_device
    if d is None:
        d = cc._draft_device = _torch().device("cuda", cc.params.device)
    return d


def _call(cc, name, args, device):
    from . import _check, lib
    stream = _torch().cuda.current_stream(device).cuda_stream
    _check(getattr(lib(), name)(cc.h, args, stream))


def _workspace(cc, name, layout, head, key, device):
    """A workspace for one call; its size is looked up once for each set of
    sizes."""
    sizes = cc._draft_sizes
    n = sizes.get((name, key))
    if n is None:
        from . import CKKSError, lib
        n = getattr(lib(), name + "_workspace")(cc.h, layout.pack(*head, 0, 0))
        if n < 0:
            raise CKKSError(1, lib().ckks_last_error().decode())
        if len(sizes) >= 256:
            sizes.clear()
        sizes[(name, key)] = n
    if n == 0:
        return None
    torch = _torch()
    return torch.empty(n, dtype=torch.uint8, device=device)


def _by_head(t):
    """(address, batch, head, row strides) of a [batch, heads, rows, ...] tensor."""
    s = t.stride()
    return t.data_ptr(), s[0], s[1], s[2]


def _by_node(t):
    """The same of a [batch, rows, heads, ...] tensor."""
    s = t.stride()
    return t.data_ptr(), s[0], s[2], s[1]


def _cache_type(t, name):
    code = _DTYPES.get(t.dtype, 3)
    if code == 3:
        _refuse(name, f"expected bfloat16, float16 or float32, got {t.dtype}")
    return code


def attention(cc, q, k_cache, v_cache, lens, k_new, v_new, parents, scale=None):
    """Attention of the drafted nodes over the cache and their ancestors.

    q [B, n, Hq, D]; k_cache, v_cache [B, Hkv, capacity, D] (the first lens[b]
    rows are used); lens [B] int32; k_new, v_new [B, n, Hkv, D]; parents [B, n]
    int32.  bfloat16, float16 or float32, Hq a multiple of Hkv, D <= 256,
    n <= 64 (one node is the single-token step), any strides with a contiguous
    last dimension.  scale defaults to 1 / sqrt(D).  Returns out [B, n, Hq, D]
    in q's type and lse [B, n, Hq] float32, the log of each row's sum.  A
    padding node's row is 0, its lse -inf."""
    torch, device = _torch(), _device(cc)
    if q.dim() != 4 or k_cache.dim() != 4:
        _refuse("q" if q.dim() != 4 else "k_cache", "expected four dimensions")
    b, n, hq, d = q.shape
    hk, cap = k_cache.shape[1], k_cache.shape[2]
    t = q.dtype
    code = _cache_type(q, "q")
    _tensor(q, "q", (b, n, hq, d), t, device)
    _tensor(k_cache, "k_cache", (b, hk, cap, d), t, device)
    _tensor(v_cache, "v_cache", (b, hk, cap, d), t, device)
    _tensor(k_new, "k_new", (b, n, hk, d), t, device)
    _tensor(v_new, "v_new", (b, n, hk, d), t, device)
    _tensor(lens, "lens", (b,), torch.int32, device, True)
    _tensor(parents, "parents", (b, n), torch.int32, device, True)
    out = torch.empty((b, n, hq, d), dtype=t, device=device)
    lse = torch.empty((b, n, hq), dtype=torch.float32, device=device)
    if b == 0:
        return out, lse
    key = (code, b, hq, hk, d, n, cap)
    head = (code, b, hq, hk, d, n, cap, 0, 1.0 / math.sqrt(d) if scale is None else float(scale), *_by_node(q),
            *_by_head(k_cache), *_by_head(v_cache), *_by_node(k_new), *_by_node(v_new), *_by_node(out),
            lens.data_ptr(), parents.data_ptr(), lse.data_ptr())
    name = "ckks_draft_attention"
    ws = _workspace(cc, name, _ATTENTION, head, key, device)
    _call(cc, name, _ATTENTION.pack(*head, ws.data_ptr() if ws is not None else 0, ws.numel() if ws is not None else 0),
          device)
    return out, lse


def verify(cc, target, draft, tokens, parents, uniforms):
    """Which drafts the target's probabilities confirm, and the next token.

    target, draft [B, n + 1, V] float32 or float64 (each its own): row 0 the
    probabilities behind the cached tokens, row i + 1 those behind node i;
    tokens, parents [B, n] int32; uniforms [B, n + 1] float64 in [0, 1).  A
    child c of the node reached, with token x, is accepted when
    uniforms[c] * q(x) < p(x); each child refused replaces p by
    max(p - q, 0) / sum; the next token is drawn from what p is at the end with
    uniforms[n].  Drafts drawn from ``draft`` give tokens distributed as
    ``target``'s.  Returns path [B, n] int32 (accepted nodes from the root on,
    then -1), count [B] int32 and token [B] int32.  Computed in float64."""
    torch, device = _torch(), _device(cc)
    if target.dim() != 3 or target.shape[1] < 1:
        _refuse("target", "expected [batch, nodes + 1, vocabulary]")
    b, n, v = target.shape[0], target.shape[1] - 1, target.shape[2]
    codes = []
    for x, name in ((target, "target"), (draft, "draft")):
        codes.append(_DTYPES.get(x.dtype, 0))
        if codes[-1] < 2:
            _refuse(name, f"expected float32 or float64, got {x.dtype}")
        _tensor(x, name, (b, n + 1, v), x.dtype, device)
    _tensor(tokens, "tokens", (b, n), torch.int32, device, True)
    _tensor(parents, "parents", (b, n), torch.int32, device, True)
    _tensor(uniforms, "uniforms", (b, n + 1), torch.float64, device, True)
    path = torch.empty((b, n), dtype=torch.int32, device=device)
    both = torch.empty((2, b), dtype=torch.int32, device=device)
    count, token = both[0], both[1]
    if b:
        ts, ds = target.stride(), draft.stride()
        _call(cc, "ckks_draft_verify", _VERIFY.pack(
            codes[0], codes[1], b, n, v, 0, target.data_ptr(), ts[0], 0, ts[1], draft.data_ptr(), ds[0], 0, ds[1],
            tokens.data_ptr(), parents.data_ptr(), uniforms.data_ptr(), path.data_ptr(), count.data_ptr(),
            token.data_ptr()), device)
    return path, count, token


def commit(cc, k_cache, v_cache, lens, k_new, v_new, path, count):
    """Appends the accepted nodes' rows to the cache (in place) and returns
    the new lengths [B] int32; arguments as for ``attention`` and as ``verify``
    returns them.  A sequence that does not fit its cache is left as it is;
    the next ``cc.Synchronize()`` behind this stream reports it."""
    torch, device = _torch(), _device(cc)
    if k_cache.dim() != 4 or k_new.dim() != 4:
        _refuse("k_cache" if k_cache.dim() != 4 else "k_new", "expected four dimensions")
    b, hk, cap, d = k_cache.shape
    n, t = k_new.shape[1], k_cache.dtype
    code = _cache_type(k_cache, "k_cache")
    for x, name in ((k_cache, "k_cache"), (v_cache, "v_cache")):
        _writable(_tensor(x, name, (b, hk, cap, d), t, device), name)
    _tensor(k_new, "k_new", (b, n, hk, d), t, device)
    _tensor(v_new, "v_new", (b, n, hk, d), t, device)
    _tensor(lens, "lens", (b,), torch.int32, device, True)
    _tensor(path, "path", (b, n), torch.int32, device, True)
    _tensor(count, "count", (b,), torch.int32, device, True)
    out = torch.empty((b,), dtype=torch.int32, device=device)
    if b:
        _call(cc, "ckks_draft_commit", _COMMIT.pack(
            code, b, hk, d, n, cap, *_by_head(k_cache), *_by_head(v_cache), *_by_node(k_new), *_by_node(v_new),
            lens.data_ptr(), path.data_ptr(), count.data_ptr(), out.data_ptr()), device)
    return out


def accumulate(cc, q, lse, k_cache, lens, path, count, acc, scale=None):
    """Adds to acc [B, Hkv, capacity] float32 (in place, returned) the
    attention weights of the accepted nodes, summed over the query heads of a
    key: q and lse as ``attention`` took and returned them, k_cache after the
    commit, lens before it.  The keys behind lens start from 0."""
    torch, device = _torch(), _device(cc)
    if q.dim() != 4 or k_cache.dim() != 4:
        _refuse("q" if q.dim() != 4 else "k_cache", "expected four dimensions")
    b, n, hq, d = q.shape
    hk, cap = k_cache.shape[1], k_cache.shape[2]
    code = _cache_type(q, "q")
    _tensor(q, "q", (b, n, hq, d), q.dtype, device)
    _tensor(k_cache, "k_cache", (b, hk, cap, d), q.dtype, device)
    _tensor(lse, "lse", (b, n, hq), torch.float32, device, True)
    _tensor(lens, "lens", (b,), torch.int32, device, True)
    _tensor(path, "path", (b, n), torch.int32, device, True)
    _tensor(count, "count", (b,), torch.int32, device, True)
    _writable(_tensor(acc, "acc", (b, hk, cap), torch.float32, device), "acc")
    if b and cap:
        s = acc.stride()
        _call(cc, "ckks_draft_accumulate", _ACCUMULATE.pack(
            code, b, hq, hk, d, n, cap, 0, 1.0 / math.sqrt(d) if scale is None else float(scale), *_by_node(q),
            *_by_head(k_cache), acc.data_ptr(), s[0], s[1], 0, lse.data_ptr(), lens.data_ptr(), path.data_ptr(),
            count.data_ptr()), device)
    return acc


def evict(cc, k_cache, v_cache, acc, lens, budget, recent, out=None):
    """Copies at most ``budget`` rows of each head's cache, in their order:
    the last ``recent`` ones and, of the others, those with the largest weights
    in acc [B, Hkv, capacity] float32 (the lower index first among equals).
    ``out``: (k, v, acc) of at least ``budget`` rows to write into, their rows
    behind the last one kept being left as they were; new tensors of exactly
    ``budget`` rows, zero behind the last one, when it is not given.  Returns
    k, v, acc, index [B, Hkv, budget] int32 (the rows kept, then -1) and the
    new lengths [B] int32."""
    torch, device = _torch(), _device(cc)
    if k_cache.dim() != 4:
        _refuse("k_cache", "expected four dimensions")
    b, hk, cap, d = k_cache.shape
    t = k_cache.dtype
    code = _cache_type(k_cache, "k_cache")
    _tensor(k_cache, "k_cache", (b, hk, cap, d), t, device)
    _tensor(v_cache, "v_cache", (b, hk, cap, d), t, device)
    _tensor(acc, "acc", (b, hk, cap), torch.float32, device)
    _tensor(lens, "lens", (b,), torch.int32, device, True)
    if budget < 1 or not 0 <= recent <= budget:
        _refuse("budget", f"need budget >= 1 and 0 <= recent <= budget, got {budget} and {recent}")
    if out is None:
        out = (torch.zeros((b, hk, budget, d), dtype=t, device=device),
               torch.zeros((b, hk, budget, d), dtype=t, device=device),
               torch.zeros((b, hk, budget), dtype=torch.float32, device=device))
    k2, v2, a2 = out
    if k2.dim() != 4:
        _refuse("out", "expected (k, v, acc) with four, four and three dimensions")
    rows = k2.shape[2]
    if rows < budget:
        _refuse("out", f"{rows} rows are fewer than the budget of {budget}")
    for x, shape, kind in ((k2, (b, hk, rows, d), t), (v2, (b, hk, rows, d), t), (a2, (b, hk, rows), torch.float32)):
        _writable(_tensor(x, "out", shape, kind, device), "out")
    index = torch.empty((b, hk, budget), dtype=torch.int32, device=device)
    new = torch.empty((b,), dtype=torch.int32, device=device)
    if b:
        s, s2 = acc.stride(), a2.stride()
        head = (code, b, hk, d, cap, rows, budget, recent, *_by_head(k_cache), *_by_head(v_cache), acc.data_ptr(),
                s[0], s[1], 0, *_by_head(k2), *_by_head(v2), a2.data_ptr(), s2[0], s2[1], 0, lens.data_ptr(),
                index.data_ptr(), new.data_ptr())
        name = "ckks_draft_evict"
        ws = _workspace(cc, name, _EVICT, head, (b, hk, cap, budget), device)
        _call(cc, name, _EVICT.pack(*head, ws.data_ptr() if ws is not None else 0, ws.numel() if ws is not None else 0),
              device)
    return k2, v2, a2, index, new
