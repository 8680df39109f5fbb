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
  draft_prompt       causal attention within packed prompts
  draft_fill         the prompts' rows appended to the cache

and over a cache in 4 bits (9/16 of a byte an element; ``row4_bytes``)
``draft_attention4``, ``draft_commit4``, ``draft_fill4`` and ``draft_read4``,
which gives its values back.

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


def prompt(cc, q, k, v, starts, scale=None):
    """Causal attention within packed prompts of different lengths.

    q [T, Hq, D]; k, v [T, Hkv, D]; starts [B + 1] int32: sequence b has the
    rows from starts[b] to starts[b + 1] (each start taken as 0..T and as no
    less than those before it).  bfloat16, float16 or float32, Hq a multiple of
    Hkv, D <= 256, any strides with a contiguous last dimension.  scale defaults
    to 1 / sqrt(D).  Returns out [T, Hq, D] in q's type and lse [T, Hq] float32,
    the log of each row's sum; a row of no sequence is 0, its lse -inf.  A
    softmax weight is rounded to the tensors' type before it meets the values.
    16-bit tensors whose rows are whole, aligned 16-byte pieces run on the tensor
    cores, others many times slower."""
    return (_binding or _native()).prompt(cc.h.value, cc.params.device, q, k, v, starts, scale)


def fill(cc, k_cache, v_cache, lens, k, v, starts):
    """Appends packed prompts' rows, k and v [T, Hkv, D] with ``starts`` as for
    ``prompt``, to the caches [B, Hkv, capacity, D] behind lens [B] int32 (in
    place) and returns the new lengths.  A sequence that does not fit its cache
    is left as it is; the next ``cc.Synchronize()`` behind this stream reports
    it."""
    return (_binding or _native()).fill(cc.h.value, cc.params.device, k_cache, v_cache, lens, k, v, starts)


def row4_bytes(head_dim):
    """Bytes of one row of a 4-bit cache: the head's elements as 4-bit floating
    point numbers (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives) in groups of
    16, behind them a scale of 8 bits for each group (a sixth of its largest
    magnitude, to three bits of mantissa), then zeros up to a multiple of four
    bytes.  A 4-bit cache is a uint8 tensor [B, Hkv, capacity, row4_bytes(D)]
    whose rows start on 4-byte boundaries; zeros are an empty one.
    ``attention4`` wants a head's rows one behind the other and 16-bit queries:
    over long caches in other orders, or in float32, it takes 15 times as
    long.  Magnitudes
    over 61440 become 61440, and a group with an infinity or a NaN in it reads
    as NaN."""
    return (_binding or _native()).row4_bytes(head_dim)


def fill4(cc, k_cache, v_cache, lens, k, v, starts):
    """``fill`` into 4-bit caches: rounds each element once, to the nearest
    number of its group's scale."""
    return (_binding or _native()).fill4(cc.h.value, cc.params.device, k_cache, v_cache, lens, k, v, starts)


def commit4(cc, k_cache, v_cache, lens, k_new, v_new, path, count):
    """``commit`` into 4-bit caches, rounded as by ``fill4``."""
    return (_binding or _native()).commit4(cc.h.value, cc.params.device, k_cache, v_cache, lens, k_new, v_new, path,
                                           count)


def read4(cc, cache, lens, head_dim, dtype):
    """The values of a 4-bit cache, [B, Hkv, capacity, head_dim] in ``dtype``
    (bfloat16, float16 or float32; each holds them exactly), 0 behind lens."""
    return (_binding or _native()).read4(cc.h.value, cc.params.device, cache, lens, head_dim, dtype)


def attention4(cc, q, k_cache, v_cache, lens, k_new, v_new, parents, scale=None):
    """``attention`` over 4-bit caches [B, Hkv, capacity, row4_bytes(D)], of
    their exact values; the new rows are in q's type."""
    return (_binding or _native()).attention4(cc.h.value, cc.params.device, q, k_cache, v_cache, lens, k_new, v_new,
                                              parents, scale)


class DraftModel:
    """The data owner's plain draft model: blocks of the weights that
    ``EncryptedBlock`` takes (bias-free pre-LN, tanh-GELU), evaluated on the
    context's GPU over a key/value cache of ``capacity`` rows per block.

    ``forward`` evaluates a tree of drafted nodes behind the cached tokens,
    ``accept`` appends the nodes that the target confirmed, ``prompt`` takes
    the packed prompts of all sequences, ``prefill`` prompts of one length in
    trees.  With ``budget``, a tree that would not fit behind the longest
    sequence's rows has every sequence cut to its ``recent`` latest and its
    heaviest keys first.  Where it might not fit, ``forward`` reads the lengths
    back (it waits for the GPU then).  With ``cache_bits=4`` the cache is kept
    in 4 bits (``row4_bytes``), without a budget: the weights that eviction
    goes by are not gathered over such a cache."""

    def __init__(self, cc, block_weights: list, capacity: int, batch: int = 1, heads: int = 12, dtype=None,
                 budget: int | None = None, recent: int = 0, cache_bits: int | None = None):
        import torch
        if cache_bits not in (None, 4):
            raise ValueError(f"cache_bits: expected 4, or None for rows of the model's type, got {cache_bits}")
        if cache_bits == 4 and budget is not None:
            raise ValueError("budget: a 4-bit cache is not cut")
        device = torch.device("cuda", cc.params.device)
        self.cc, self.heads, self.batch, self.capacity = cc, heads, batch, capacity
        self.budget, self.recent, self._four = budget, recent, cache_bits == 4
        self.dtype = torch.bfloat16 if dtype is None else dtype
        if budget is not None and budget + MAX_NODES > capacity:
            raise ValueError(f"budget: {budget} rows and a tree of {MAX_NODES} nodes do not fit a capacity of {capacity}")
        names = ("ln1", "attn_qkv", "attn_proj", "ln2", "mlp_fc", "mlp_proj")
        self.weights = [{k: torch.as_tensor(w[k]).to(device=device, dtype=torch.float32 if k[:2] == "ln" else self.dtype)
                         for k in names} for w in block_weights]
        self.width = self.weights[0]["ln1"].shape[0]

        def caches():
            size = self.width // heads
            rows, kind = (batch, heads, capacity, row4_bytes(size) if self._four else size), \
                torch.uint8 if self._four else self.dtype
            # (keys, values, the keys' weights: none over 4-bit rows, which are not cut)
            return [(torch.zeros(rows, dtype=kind, device=device), torch.zeros(rows, dtype=kind, device=device),
                     None if self._four else torch.zeros(rows[:3], device=device)) for _ in block_weights]

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
        x, steps, attend = x.to(torch.float32), [], attention4 if self._four else attention
        for w, (k_cache, v_cache, _) in zip(self.weights, self.caches):
            q, k, v = self._qkv(x, w).view(b, n, 3, self.heads, width // self.heads).unbind(2)
            out, lse = attend(self.cc, q, k_cache, v_cache, self.lens, k, v, parents)
            x = self._rest(x, out.reshape(b, n, width), w)
            steps.append((q, lse, k, v))
        self._steps = steps
        return x

    def _qkv(self, x, w):
        import torch
        return torch.layer_norm(x, (self.width,), w["ln1"], None, 1e-5).to(self.dtype) @ w["attn_qkv"].T

    def _rest(self, x, out, w):
        """A block behind its attention."""
        import torch
        x = x + (out @ w["attn_proj"].T).float()
        h = torch.layer_norm(x, (self.width,), w["ln2"], None, 1e-5).to(self.dtype)
        h = torch.nn.functional.gelu(h @ w["mlp_fc"].T, approximate="tanh")
        return x + (h @ w["mlp_proj"].T).float()

    def accept(self, path, count):
        """Appends the nodes path[:, :count] of the last ``forward`` to every
        block's cache, and their attention weights to its keys'."""
        if self._steps is None:
            raise RuntimeError("accept follows a forward")
        lens, append = self.lens, commit4 if self._four else commit
        for (q, lse, k, v), (k_cache, v_cache, acc) in zip(self._steps, self.caches):
            self.lens = append(self.cc, k_cache, v_cache, lens, k, v, path, count)
            if self.budget is not None:
                accumulate(self.cc, q, lse, k_cache, lens, path, count, acc)
        self._most = min(self.capacity, self._most + path.shape[1])
        self._steps = None

    def prompt(self, x, starts):
        """The sequences' prompts, packed: embeddings x [T, D], starts
        [batch + 1] int32 as for ``drafting.prompt``.  Returns the hidden states
        [T, D] (float32).  The caches must be empty, and hold the longest prompt
        (``starts`` is read back where the rows might be more than the
        capacity, the lengths where the caches were in use: ``lens.zero_()``
        empties them for the next prompts).  A model with a budget takes its prompt through ``prefill``,
        which gathers the weights that eviction goes by."""
        import torch
        if self.budget is not None:
            raise ValueError("prompt: a model with a budget gathers its prompt's weights through prefill")
        if self._most and self.lens.any():  # `_most` may count rows that were never accepted, or are gone
            raise ValueError("prompt: the cache holds rows already")
        t, width = x.shape
        most = t
        if t > self.capacity:
            s = starts.clamp(0, t).cummax(0).values
            most = int((s[1:] - s[:-1]).max())
            if most > self.capacity:
                raise ValueError(f"a prompt of {most} tokens exceeds the capacity of {self.capacity}")
        x, lens, append = x.to(torch.float32), self.lens, fill4 if self._four else fill
        for w, (k_cache, v_cache, _) in zip(self.weights, self.caches):
            q, k, v = self._qkv(x, w).view(t, 3, self.heads, width // self.heads).unbind(1)
            out, _ = prompt(self.cc, q, k, v, starts)
            self.lens = append(self.cc, k_cache, v_cache, lens, k, v, starts)
            x = self._rest(x, out.reshape(t, width), w)
        self._most, self._steps = most, None
        return x

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
