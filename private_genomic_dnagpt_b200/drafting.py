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


_entries: dict = {}  # the library's entry points by name, looked up once
_current_stream = None


def _torch():
    import torch
    global _current_stream
    if not _DTYPES:
        _DTYPES.update({torch.bfloat16: 0, torch.float16: 1, torch.float32: 2, torch.float64: 3})
        # the handle of torch's current stream, without a Stream object where torch offers that
        _current_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
            lambda index: torch.cuda.current_stream(index).cuda_stream)
    return torch


def _refuse(name, why):
    raise ValueError(f"{name}: {why}")


def _complain(t, name, shape, dtype, device, small):
    """Says what is wrong with an argument that did not pass."""
    if not isinstance(t, _torch().Tensor):
        _refuse(name, f"expected a tensor, got {type(t).__name__}")
    if t.shape != shape:
        _refuse(name, f"expected the shape {tuple(shape)}, got {tuple(t.shape)}")
    if t.dtype is not dtype:
        _refuse(name, f"expected {dtype}, got {t.dtype}")
    if t.device != device:
        _refuse(name, f"expected a tensor of {device}, the context's device, got {t.device}")
    if t.requires_grad and _torch().is_grad_enabled():
        _refuse(name, "requires a gradient, which this operator does not have (call it under torch.no_grad)")
    _refuse(name, "must be contiguous" if small else "its last dimension must be contiguous")


# The checks of a call take about as long as its launch, so each tensor's
# attributes are read once: _strides and _small return what the packed
# arguments need.

def _strides(t, name, shape, dtype, device, where, grad):
    """Checks a tensor of rows and returns its strides."""
    if t.shape != shape or t.dtype is not dtype or t.get_device() != where or (grad and t.requires_grad):
        _complain(t, name, shape, dtype, device, False)
    s = t.stride()
    if s[-1] != 1 and shape[-1] > 1 and t.numel():
        _complain(t, name, shape, dtype, device, False)
    return s


def _small(t, name, shape, dtype, device, where, grad):
    """Checks a contiguous tensor and returns its address."""
    if (t.shape != shape or t.dtype is not dtype or t.get_device() != where or not t.is_contiguous()
            or (grad and t.requires_grad)):
        _complain(t, name, shape, dtype, device, True)
    return t.data_ptr()


def _writable(name, shape, strides):
    """Refuses a tensor of which two elements share memory."""
    if 0 in strides:
        for n, s in zip(shape, strides):
            if n > 1 and s == 0:
                _refuse(name, "is written, but some of its elements share memory")


def _setting(cc):
    """torch, the context's device, its index and whether gradients are on."""
    torch = _torch()
    d = cc._draft_device
    if d is None:
        d = cc._draft_device = torch.device("cuda", cc.params.device)
    return torch, d, -1 if d.index is None else d.index, torch.is_grad_enabled()


def _call(cc, name, args, where):
    f = _entries.get(name)
    if f is None:
        from . import lib
        f = _entries[name] = getattr(lib(), name)
    rc = f(cc.h, args, _current_stream(where))
    if rc:
        from . import _check
        _check(rc)


def _workspace(cc, name, layout, head, key, device):
    """A workspace for one call; its size is looked up once for each set of
    sizes."""
    sizes = cc._draft_sizes
    n = sizes.get(key)
    if n is None:
        from . import CKKSError, lib
        n = getattr(lib(), name + "_workspace")(cc.h, layout.pack(*head, 0, 0))
        if n < 0:
            raise CKKSError(1, lib().ckks_last_error().decode())
        if len(sizes) >= 256:
            sizes.clear()
        sizes[key] = n
    if n == 0:
        return None
    torch = _torch()
    return torch.empty(n, dtype=torch.uint8, device=device)


def _four(t, name):
    if t.dim() != 4:
        _refuse(name, "expected four dimensions")
    return t.shape


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
    torch, device, where, grad = _setting(cc)
    shape, cache = _four(q, "q"), _four(k_cache, "k_cache")
    b, n, hq, d = shape
    hk, cap = cache[1], cache[2]
    t, code = q.dtype, _cache_type(q, "q")
    rows, rest, new, i32 = (b, hk, cap, d), (t, device, where, grad), (b, n, hk, d), torch.int32
    sq = _strides(q, "q", shape, *rest)
    sk, sv = _strides(k_cache, "k_cache", rows, *rest), _strides(v_cache, "v_cache", rows, *rest)
    nk, nv = _strides(k_new, "k_new", new, *rest), _strides(v_new, "v_new", new, *rest)
    len_at = _small(lens, "lens", (b,), i32, device, where, grad)
    parents_at = _small(parents, "parents", (b, n), i32, device, where, grad)
    out = q.new_empty(shape)
    lse = q.new_empty((b, n, hq), dtype=torch.float32)
    if b == 0:
        return out, lse
    key = ("attention", code, b, hq, hk, d, n, cap)
    row = hq * d
    head = (code, b, hq, hk, d, n, cap, 0, 1.0 / math.sqrt(d) if scale is None else float(scale),
            q.data_ptr(), sq[0], sq[2], sq[1], k_cache.data_ptr(), sk[0], sk[1], sk[2],
            v_cache.data_ptr(), sv[0], sv[1], sv[2], k_new.data_ptr(), nk[0], nk[2], nk[1],
            v_new.data_ptr(), nv[0], nv[2], nv[1], out.data_ptr(), n * row, d, row, len_at, parents_at, lse.data_ptr())
    ws = _workspace(cc, "ckks_draft_attention", _ATTENTION, head, key, device)
    args = _ATTENTION.pack(*head, 0, 0) if ws is None else _ATTENTION.pack(*head, ws.data_ptr(), ws.numel())
    _call(cc, "ckks_draft_attention", args, where)
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
    torch, device, where, grad = _setting(cc)
    if target.dim() != 3 or target.shape[1] < 1:
        _refuse("target", "expected [batch, nodes + 1, vocabulary]")
    shape = target.shape
    b, n, v = shape[0], shape[1] - 1, shape[2]
    tc, dc = _DTYPES.get(target.dtype, 0), _DTYPES.get(draft.dtype, 0)
    for code, x, name in ((tc, target, "target"), (dc, draft, "draft")):
        if code < 2:
            _refuse(name, f"expected float32 or float64, got {x.dtype}")
    ts = _strides(target, "target", shape, target.dtype, device, where, grad)
    ds = _strides(draft, "draft", shape, draft.dtype, device, where, grad)
    rest = (torch.int32, device, where, grad)
    tokens_at, parents_at = _small(tokens, "tokens", (b, n), *rest), _small(parents, "parents", (b, n), *rest)
    uniforms_at = _small(uniforms, "uniforms", (b, n + 1), torch.float64, device, where, grad)
    path, both = torch.empty_like(tokens), tokens.new_empty((2, b))
    count, token = both.unbind()
    if b:
        at = both.data_ptr()
        _call(cc, "ckks_draft_verify", _VERIFY.pack(
            tc, dc, b, n, v, 0, target.data_ptr(), ts[0], 0, ts[1], draft.data_ptr(), ds[0], 0, ds[1],
            tokens_at, parents_at, uniforms_at, path.data_ptr(), at, at + 4 * b), where)
    return path, count, token


def commit(cc, k_cache, v_cache, lens, k_new, v_new, path, count):
    """Appends the accepted nodes' rows to the cache (in place) and returns
    the new lengths [B] int32; arguments as for ``attention`` and as ``verify``
    returns them.  A sequence that does not fit its cache is left as it is;
    the next ``cc.Synchronize()`` behind this stream reports it."""
    torch, device, where, grad = _setting(cc)
    rows, new = _four(k_cache, "k_cache"), _four(k_new, "k_new")
    b, hk, cap, d = rows
    n, t, code = new[1], k_cache.dtype, _cache_type(k_cache, "k_cache")
    rest, new, ints = (t, device, where, grad), (b, n, hk, d), (torch.int32, device, where, grad)
    sk, sv = _strides(k_cache, "k_cache", rows, *rest), _strides(v_cache, "v_cache", rows, *rest)
    _writable("k_cache", rows, sk)
    _writable("v_cache", rows, sv)
    nk, nv = _strides(k_new, "k_new", new, *rest), _strides(v_new, "v_new", new, *rest)
    len_at, path_at = _small(lens, "lens", (b,), *ints), _small(path, "path", (b, n), *ints)
    count_at = _small(count, "count", (b,), *ints)
    out = torch.empty_like(lens)
    if b:
        _call(cc, "ckks_draft_commit", _COMMIT.pack(
            code, b, hk, d, n, cap, k_cache.data_ptr(), sk[0], sk[1], sk[2], v_cache.data_ptr(), sv[0], sv[1], sv[2],
            k_new.data_ptr(), nk[0], nk[2], nk[1], v_new.data_ptr(), nv[0], nv[2], nv[1],
            len_at, path_at, count_at, out.data_ptr()), where)
    return out


def accumulate(cc, q, lse, k_cache, lens, path, count, acc, scale=None):
    """Adds to acc [B, Hkv, capacity] float32 (in place, returned) the
    attention weights of the accepted nodes, summed over the query heads of a
    key: q and lse as ``attention`` took and returned them, k_cache after the
    commit, lens before it.  The keys behind lens start from 0."""
    torch, device, where, grad = _setting(cc)
    shape, cache = _four(q, "q"), _four(k_cache, "k_cache")
    b, n, hq, d = shape
    hk, cap = cache[1], cache[2]
    code = _cache_type(q, "q")
    ints = (torch.int32, device, where, grad)
    sq = _strides(q, "q", shape, q.dtype, device, where, grad)
    sk = _strides(k_cache, "k_cache", (b, hk, cap, d), q.dtype, device, where, grad)
    lse_at = _small(lse, "lse", (b, n, hq), torch.float32, device, where, grad)
    len_at, path_at = _small(lens, "lens", (b,), *ints), _small(path, "path", (b, n), *ints)
    count_at = _small(count, "count", (b,), *ints)
    sa = _strides(acc, "acc", (b, hk, cap), torch.float32, device, where, grad)
    _writable("acc", (b, hk, cap), sa)
    if b and cap:
        _call(cc, "ckks_draft_accumulate", _ACCUMULATE.pack(
            code, b, hq, hk, d, n, cap, 0, 1.0 / math.sqrt(d) if scale is None else float(scale),
            q.data_ptr(), sq[0], sq[2], sq[1], k_cache.data_ptr(), sk[0], sk[1], sk[2], acc.data_ptr(), sa[0], sa[1], 0,
            lse_at, len_at, path_at, count_at), where)
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
    torch, device, where, grad = _setting(cc)
    rows = _four(k_cache, "k_cache")
    b, hk, cap, d = rows
    t, code, f32 = k_cache.dtype, _cache_type(k_cache, "k_cache"), torch.float32
    rest = (device, where, grad)
    sk, sv = _strides(k_cache, "k_cache", rows, t, *rest), _strides(v_cache, "v_cache", rows, t, *rest)
    sa = _strides(acc, "acc", (b, hk, cap), f32, *rest)
    len_at = _small(lens, "lens", (b,), torch.int32, *rest)
    if budget < 1 or not 0 <= recent <= budget:
        _refuse("budget", f"need budget >= 1 and 0 <= recent <= budget, got {budget} and {recent}")
    if out is None:
        out = (torch.zeros((b, hk, budget, d), dtype=t, device=device),
               torch.zeros((b, hk, budget, d), dtype=t, device=device),
               torch.zeros((b, hk, budget), dtype=f32, device=device))
    k2, v2, a2 = out
    kept = _four(k2, "out")[2]
    if kept < budget:
        _refuse("out", f"{kept} rows are fewer than the budget of {budget}")
    sk2, sv2 = _strides(k2, "out", (b, hk, kept, d), t, *rest), _strides(v2, "out", (b, hk, kept, d), t, *rest)
    sa2 = _strides(a2, "out", (b, hk, kept), f32, *rest)
    _writable("out", (b, hk, kept, d), sk2)
    _writable("out", (b, hk, kept, d), sv2)
    _writable("out", (b, hk, kept), sa2)
    index, new = lens.new_empty((b, hk, budget)), torch.empty_like(lens)
    if b:
        head = (code, b, hk, d, cap, kept, budget, recent, k_cache.data_ptr(), sk[0], sk[1], sk[2],
                v_cache.data_ptr(), sv[0], sv[1], sv[2], acc.data_ptr(), sa[0], sa[1], 0,
                k2.data_ptr(), sk2[0], sk2[1], sk2[2], v2.data_ptr(), sv2[0], sv2[1], sv2[2],
                a2.data_ptr(), sa2[0], sa2[1], 0, len_at, index.data_ptr(), new.data_ptr())
        ws = _workspace(cc, "ckks_draft_evict", _EVICT, head, ("evict", b, hk, cap, budget), device)
        args = _EVICT.pack(*head, 0, 0) if ws is None else _EVICT.pack(*head, ws.data_ptr(), ws.numel())
        _call(cc, "ckks_draft_evict", args, where)
    return k2, v2, a2, index, new


class DraftModel:
    """The data owner's plain draft model: blocks of the weights that
    ``EncryptedBlock`` takes (bias-free pre-LN, tanh-GELU), evaluated on the
    context's GPU over a key/value cache of ``capacity`` rows per block.

    ``forward`` evaluates a tree of drafted nodes behind the cached tokens,
    ``accept`` appends the nodes that the target confirmed, ``prefill`` takes
    a prompt.  With ``budget``, the cache is cut to its ``recent`` latest and
    its heaviest keys before it would overflow."""

    def __init__(self, cc, block_weights: list, capacity: int, batch: int = 1, heads: int = 12, dtype=None,
                 budget: int | None = None, recent: int = 0):
        torch, device, _, _ = _setting(cc)
        self.cc, self.heads, self.batch, self.capacity = cc, heads, batch, capacity
        self.budget, self.recent = budget, recent
        self.dtype = torch.bfloat16 if dtype is None else dtype
        if budget is not None and budget + MAX_NODES > capacity:
            _refuse("budget", f"{budget} rows and a tree of {MAX_NODES} nodes do not fit a capacity of {capacity}")
        names = ("ln1", "attn_qkv", "attn_proj", "ln2", "mlp_fc", "mlp_proj")
        self.weights = [{k: torch.as_tensor(w[k]).to(device=device, dtype=torch.float32 if k[:2] == "ln" else self.dtype)
                         for k in names} for w in block_weights]
        self.width = self.weights[0]["ln1"].shape[0]

        def caches():
            rows = (batch, heads, capacity, self.width // heads)
            return [(torch.zeros(rows, dtype=self.dtype, device=device), torch.zeros(rows, dtype=self.dtype, device=device),
                     torch.zeros(rows[:3], device=device)) for _ in block_weights]

        self.caches, self._spare = caches(), caches() if budget is not None else None
        self.lens = torch.zeros(batch, dtype=torch.int32, device=device)
        self._most = 0  # no sequence has more rows than this
        self._steps = None

    def forward(self, x, parents):
        """Hidden states [batch, n, D] (float32) of the nodes with embeddings
        x [batch, n, D] and parents [batch, n] int32 behind the cached tokens.
        The nodes' rows are kept for ``accept``."""
        torch = _torch()
        b, n, width = x.shape
        if self._most + n > self.capacity:
            self._make_room(n)
        x, steps = x.to(torch.float32), []
        for w, (k_cache, v_cache, _) in zip(self.weights, self.caches):
            h = torch.layer_norm(x, (width,), w["ln1"], None, 1e-5).to(self.dtype)
            q, k, v = (h @ w["attn_qkv"].T).view(b, n, 3, self.heads, width // self.heads).unbind(2)
            out, lse = attention(self.cc, q, k_cache, v_cache, self.lens, k, v, parents)
            x = x + (out.reshape(b, n, width) @ w["attn_proj"].T).float()
            h = torch.layer_norm(x, (width,), w["ln2"], None, 1e-5).to(self.dtype)
            h = torch.nn.functional.gelu(h @ w["mlp_fc"].T, approximate="tanh")
            x = x + (h @ w["mlp_proj"].T).float()
            steps.append((q, lse, k, v))
        self._steps = steps
        return x

    def accept(self, path, count):
        """Appends the nodes path[:, :count] of the last ``forward`` to every
        block's cache, and their attention weights to its keys'."""
        if self._steps is None:
            raise RuntimeError("accept follows a forward")
        lens = self.lens
        for (q, lse, k, v), (k_cache, v_cache, acc) in zip(self._steps, self.caches):
            self.lens = commit(self.cc, k_cache, v_cache, lens, k, v, path, count)
            if self.budget is not None:
                accumulate(self.cc, q, lse, k_cache, lens, path, count, acc)
        self._most = min(self.capacity, self._most + path.shape[1])
        self._steps = None

    def prefill(self, x):
        """A prompt's embeddings [batch, m, D], in chains of 64 nodes; returns
        the hidden states [batch, m, D]."""
        torch = _torch()
        got = []
        for c in x.split(MAX_NODES, dim=1):
            n = c.shape[1]
            chain = torch.arange(n, dtype=torch.int32, device=c.device).repeat(self.batch, 1)
            got.append(self.forward(c, chain - 1))
            self.accept(chain, torch.full((self.batch,), n, dtype=torch.int32, device=c.device))
        return torch.cat(got, 1)

    def _make_room(self, n):
        """Before n more rows: the cache cut to its budget, or, without one,
        the rows counted exactly."""
        if self.budget is None:
            self._most = int(self.lens.max())
            if self._most + n > self.capacity:
                raise ValueError(f"{self._most} cached rows and {n} nodes exceed the capacity of {self.capacity}")
            return
        lens = self.lens
        for i, (k, v, acc) in enumerate(self.caches):
            _, _, _, _, self.lens = evict(self.cc, k, v, acc, lens, self.budget, self.recent, out=self._spare[i])
        self.caches, self._spare = self._spare, self.caches
        self._most = min(self._most, self.budget)
