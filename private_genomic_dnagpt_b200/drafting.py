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

MAX_NODES = 64  # nodes of one tree

_binding = None


def _native():
    """The compiled binding (csrc/torch_draft.cpp), built on its first use
    where it is absent."""
    global _binding
    if _binding is None:
        import importlib.util
        import os

        import torch  # noqa: F401  (the binding links against its libraries)

        from . import lib
        lib()
        path = os.path.join(os.path.dirname(os.path.abspath(__file__)), "_draft.so")
        if not os.path.exists(path):
            from .build import build_binding
            build_binding()
        spec = importlib.util.spec_from_file_location(__package__ + "._draft", path)
        _binding = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(_binding)
    return _binding


def attention(cc, q, k_cache, v_cache, lens, k_new, v_new, parents, scale=None):
    """Attention of the drafted nodes over the cache and their ancestors.

    q [B, n, Hq, D]; k_cache, v_cache [B, Hkv, capacity, D] (the first lens[b]
    rows are used); lens [B] int32; k_new, v_new [B, n, Hkv, D]; parents [B, n]
    int32.  bfloat16, float16 or float32, Hq a multiple of Hkv, D <= 256,
    n <= 64 (one node is the single-token step), any strides with a contiguous
    last dimension.  scale defaults to 1 / sqrt(D).  Returns out [B, n, Hq, D]
    in q's type and lse [B, n, Hq] float32, the log of each row's sum.  A
    padding node's row is 0, its lse -inf."""
    return (_binding or _native()).attention(cc.h.value, cc.params.device, q, k_cache, v_cache, lens, k_new, v_new,
                                             parents, scale)


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
    return (_binding or _native()).verify(cc.h.value, cc.params.device, target, draft, tokens, parents, uniforms)


def commit(cc, k_cache, v_cache, lens, k_new, v_new, path, count):
    """Appends the accepted nodes' rows to the cache (in place) and returns
    the new lengths [B] int32; arguments as for ``attention`` and as ``verify``
    returns them.  A sequence that does not fit its cache is left as it is;
    the next ``cc.Synchronize()`` behind this stream reports it."""
    return (_binding or _native()).commit(cc.h.value, cc.params.device, k_cache, v_cache, lens, k_new, v_new, path, count)


def accumulate(cc, q, lse, k_cache, lens, path, count, acc, scale=None):
    """Adds to acc [B, Hkv, capacity] float32 (in place, returned) the
    attention weights of the accepted nodes, summed over the query heads of a
    key: q and lse as ``attention`` took and returned them, k_cache after the
    commit, lens before it.  The keys behind lens start from 0."""
    return (_binding or _native()).accumulate(cc.h.value, cc.params.device, q, lse, k_cache, lens, path, count, acc,
                                              scale)


def evict(cc, k_cache, v_cache, acc, lens, budget, recent, out=None):
    """Copies at most ``budget`` rows of each head's cache, in their order:
    the last ``recent`` ones and, of the others, those with the largest weights
    in acc [B, Hkv, capacity] float32 (the lower index first among equals, a
    weight that is not a number behind all others).
    ``out``: (k, v, acc) of at least ``budget`` rows to write into, their rows
    behind the last one kept being left as they were; new tensors of exactly
    ``budget`` rows, zero behind the last one, when it is not given.  Returns
    k, v, acc, index [B, Hkv, budget] int32 (the rows kept, then -1) and the
    new lengths [B] int32."""
    return (_binding or _native()).evict(cc.h.value, cc.params.device, k_cache, v_cache, acc, lens, budget, recent, out)


class DraftModel:
    """The data owner's plain draft model: blocks of the weights that
    ``EncryptedBlock`` takes (bias-free pre-LN, tanh-GELU), evaluated on the
    context's GPU over a key/value cache of ``capacity`` rows per block.

    ``forward`` evaluates a tree of drafted nodes behind the cached tokens,
    ``accept`` appends the nodes that the target confirmed, ``prefill`` takes
    a prompt.  With ``budget``, a tree that would not fit behind the longest
    sequence's rows has every sequence cut to its ``recent`` latest and its
    heaviest keys first.  Where it might not fit, ``forward`` reads the lengths
    back (it waits for the GPU then)."""

    def __init__(self, cc, block_weights: list, capacity: int, batch: int = 1, heads: int = 12, dtype=None,
                 budget: int | None = None, recent: int = 0):
        import torch
        device = torch.device("cuda", cc.params.device)
        self.cc, self.heads, self.batch, self.capacity = cc, heads, batch, capacity
        self.budget, self.recent = budget, recent
        self.dtype = torch.bfloat16 if dtype is None else dtype
        if budget is not None and budget + MAX_NODES > capacity:
            raise ValueError(f"budget: {budget} rows and a tree of {MAX_NODES} nodes do not fit a capacity of {capacity}")
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
        import torch
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
        import torch
        got = []
        for c in x.split(MAX_NODES, dim=1):
            n = c.shape[1]
            chain = torch.arange(n, dtype=torch.int32, device=c.device).repeat(self.batch, 1)
            got.append(self.forward(c, chain - 1))
            self.accept(chain, torch.full((self.batch,), n, dtype=torch.int32, device=c.device))
        return torch.cat(got, 1)

    def _make_room(self, n):
        """Before n more rows than `_most` leaves room for: the rows counted
        exactly (`accept` only knows how many there are at most) and, where
        they would not fit, the cache cut to its budget."""
        self._most = int(self.lens.max())
        if self._most + n <= self.capacity:
            return
        if self.budget is None:
            raise ValueError(f"{self._most} cached rows and {n} nodes exceed the capacity of {self.capacity}")
        lens = self.lens
        for i, (k, v, acc) in enumerate(self.caches):
            _, _, _, _, self.lens = evict(self.cc, k, v, acc, lens, self.budget, self.recent, out=self._spare[i])
        self.caches, self._spare = self._spare, self.caches
        self._most = min(self._most, self.budget)
