"""Prompts and 4-bit caches of the data owner's draft model, as measured cases.

Before the data owner drafts its first token, its draft model takes the prompts
of all sequences that are served; behind them it keeps keys and values, which
hold nine sixteenths of a byte an element in 4 bits:

  prompt   causal attention within packed prompts of different lengths
  fill     the prompts' keys and values written to a 4-bit cache, which is then
           read back
  commit   the accepted nodes of a tree of drafts written to it, and read back
  attend   attention of a tree of drafted tokens over a 4-bit cache (one node
           is the single-token decode step)

A row of a 4-bit cache is the head's elements in groups of 16: each element a
4-bit floating-point number (sign, two exponent bits, one mantissa bit: 0, 0.5,
1, 1.5, 2, 3, 4, 6), each group an 8-bit scale (five exponent bits, three of
mantissa, no sign).  It holds the groups' elements, 8 bytes each with the even
element in a byte's low half, then the groups' scales, and zeros up to a
multiple of four bytes.

``run`` is the plain form in torch when ``own`` is false, and the calls of this
repository's ``CryptoContext`` when it is true.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
DEVICE = "cuda"
VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
TOP = 10240.0  # the largest scale: six of it are a float16

_context = []


def context():
    """The context that a program keeps: one small ring, no keys needed."""
    if not _context:
        import private_genomic_dnagpt_b200 as eng
        _context.append(eng.GenCryptoContext(eng.CCParams(ring_dim_log=10, limbs=3, dnum=1, seed=1)))
    return _context[0]


# ---- the cases ---------------------------------------------------------------

def listed():
    return [
        # one prompt of the model's own length, 12 heads of 64: latency
        dict(name="prompt of 103 tokens", op="prompt", dtype="bf16", batch=1, q_heads=12, kv_heads=12, head_dim=64,
             length=103, spare=0),
        # a served batch of prompts, the longest of 2001 tokens, one token and none among them, packed into a buffer
        # that is a little longer
        dict(name="packed prompts to 2001", op="prompt", dtype="fp16", batch=12, q_heads=12, kv_heads=12, head_dim=64,
             length=2001, spare=37),
        # a long genomic context and a draft model with shared key/value heads
        dict(name="prompt of 8192", op="prompt", dtype="bf16", batch=1, q_heads=32, kv_heads=8, head_dim=128,
             length=8192, spare=0),
        # a draft model kept in 32 bits
        dict(name="prompts to 1030, fp32", op="prompt", dtype="fp32", batch=4, q_heads=12, kv_heads=12, head_dim=64,
             length=1030, spare=0),
        # the keys and values of one layer for one prompt
        dict(name="fill with 103 tokens", op="fill", dtype="bf16", batch=1, kv_heads=12, head_dim=64, length=103,
             cached=0),
        # and for a batch of long ones, behind a shared prefix that is cached already
        dict(name="fill with prompts to 8001", op="fill", dtype="bf16", batch=8, kv_heads=8, head_dim=128, length=8001,
             cached=64),
        # a served batch after a round of drafting
        dict(name="commit from trees of 31", op="commit", dtype="fp16", batch=16, nodes=31, branch=2, kv_heads=12,
             head_dim=64, length=500, accepted=4),
        # one layer's cache after a chain of drafts: launches
        dict(name="commit a chain of 5", op="commit", dtype="bf16", batch=1, nodes=5, branch=1, kv_heads=12,
             head_dim=64, length=103, accepted=3),
        # the draft model's next token behind a prompt of 103 tokens; latency
        dict(name="attend one node, 103 keys", op="attend", dtype="bf16", batch=1, nodes=1, branch=1, q_heads=12,
             kv_heads=12, head_dim=64, length=103, ragged=False),
        # eight sequences, each a binary tree of 21 drafts over a context of some thousand tokens, padded batch
        dict(name="attend trees of 21, 4001 keys", op="attend", dtype="fp16", batch=8, nodes=21, branch=2, q_heads=12,
             kv_heads=12, head_dim=64, length=4001, ragged=True),
        # single-token steps over long contexts, 4 query heads on each key/value head
        dict(name="attend one node, 65536 keys", op="attend", dtype="bf16", batch=4, nodes=1, branch=1, q_heads=32,
             kv_heads=8, head_dim=128, length=65536, ragged=False),
        # and trees over them
        dict(name="attend trees of 16, 32768 keys", op="attend", dtype="bf16", batch=2, nodes=16, branch=3, q_heads=32,
             kv_heads=8, head_dim=128, length=32768, ragged=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49))))))


def draw(rng):
    op = rng.choice(["prompt", "prompt", "fill", "commit", "attend", "attend"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    kv_heads, head_dim = rng.choice([1, 2, 4, 8, 12, 16]), rng.choice([32, 64, 64, 80, 96, 100, 128, 128, 256])
    c = dict(op=op, dtype=dtype, batch=_log(rng, 1, 16), kv_heads=kv_heads, head_dim=head_dim, length=1)
    if op == "prompt":
        c["q_heads"] = kv_heads * rng.choice([1, 1, 2, 4])
        # at most 2^28 scores of a padded batch (the largest listed case has eight times that)
        most = math.isqrt((1 << 28) // (c["batch"] * c["q_heads"]))
        c["length"], c["spare"] = _log(rng, 1, min(8192, most)), rng.choice([0, 0, rng.randint(1, 100)])
        return c
    # at most 2^25 values in the keys
    c["length"] = _log(rng, 1, max(2, min(65536, (1 << 25) // (c["batch"] * kv_heads * head_dim))))
    if op == "fill":
        c["cached"] = rng.choice([0, 0, rng.randint(1, 200)])
        return c
    c["nodes"], c["branch"] = _log(rng, 1, 64), rng.randint(1, 4)
    if op == "attend":
        c["q_heads"] = kv_heads * rng.choice([1, 1, 2, 4] if c["nodes"] <= 32 else [1, 1, 2])
        c["ragged"] = rng.random() < 0.5
    else:
        c["accepted"] = rng.randint(1, 8)
    return c


def lengths(c):
    """Tokens of each sequence: the whole length down to half of it; of a large batch the last two have one and none."""
    n, b = c["length"], c["batch"]
    got = [n - (n // 2) * i // b for i in range(b)]
    if b >= 6:
        got[-2:] = [1, 0]
    return got


def nodes_of(c):
    """Nodes of each sequence's tree; the rest of its row is padding."""
    return [max(1, c["nodes"] - (i % 3 if c.get("ragged") else 0)) for i in range(c["batch"])]


def depth_sum(c, n):
    """Keys of the tree that its n nodes see, each node its own among them."""
    d = []
    for i in range(n):
        p = i // c["branch"] - 1
        d.append(1 + (d[p] if p >= 0 else 0))
    return sum(d)


def path_of(c):
    """The first child of each node, from the root on: at most `accepted` nodes."""
    got, i = [], 0
    while i < c["nodes"] and len(got) < c["accepted"]:
        got.append(i)
        i = c["branch"] * (i + 1)
    return got


def counts(c):
    """Accepted nodes of each sequence: every third one accepted one less."""
    a = len(path_of(c))
    return [max(0, a - (i % 3 == 2)) for i in range(c["batch"])]


def row_bytes(d):
    """Bytes of one row of a 4-bit cache."""
    return -(-9 * -(-d // 16) // 4) * 4


def capacity(c):
    return c["length"] + c.get("nodes", 0) + c.get("cached", 0)


def work(c):
    e, b, op, d, hk = BYTES[c["dtype"]], c["batch"], c["op"], c["head_dim"], c["kv_heads"]
    r = row_bytes(d)
    if op == "prompt":
        t, hq = sum(lengths(c)) + c["spare"], c["q_heads"]
        return {"bytes": e * d * 2 * (hq + hk) * t + 4 * hq * t, "flops": 2 * hq * d * sum(n * (n + 1) for n in lengths(c))}
    if op in ("fill", "commit"):
        new = sum(lengths(c)) if op == "fill" else sum(counts(c))
        held = new + (b * c["cached"] if op == "fill" else sum(lengths(c)))
        # written, then read back as the type, zeros behind the last row
        return {"bytes": 2 * hk * (new * (e * d + r) + held * r + b * capacity(c) * e * d), "flops": 0}
    hq, n = c["q_heads"], c["nodes"]
    seen = sum(m * s + depth_sum(c, m) for m, s in zip(nodes_of(c), lengths(c)))
    return {"bytes": 2 * hk * (r * sum(lengths(c)) + e * d * sum(nodes_of(c))) + b * n * hq * (2 * e * d + 4),
            "flops": 4 * hq * d * seen}


# ---- a 4-bit cache's rows ------------------------------------------------------

def pack(x):
    """[..., d] of any type as rows of 4-bit numbers, [..., row_bytes(d)] uint8: the scale a sixth of the group's
    largest magnitude, rounded to three bits of mantissa (2^-17 at the finest, TOP at most), each element the nearest
    4-bit number of it, both to even in the middle.  A group with an infinity or no number in it has the scale 0xFC, no
    number."""
    d = x.shape[-1]
    x = torch.nn.functional.pad(x.float(), (0, -d % 16))
    x = x.unflatten(-1, (-(-d // 16), 16))
    top = x.abs().amax(-1)
    fine = torch.isfinite(x).all(-1)
    # in 64 bits: values next to the border between two of fewer bits
    a = torch.where(fine, top, 0.0).double() / 6
    step = torch.exp2((torch.frexp(a).exponent - 1).clamp(min=-14).double() - 3)
    s = (torch.round(a / step) * step).clamp(max=TOP)
    y = x.abs().double() / torch.where(s > 0, s, 1.0)[..., None]
    y = torch.where((fine & (s > 0))[..., None], y, 0.0)
    code = ((y > 0.25).to(torch.uint8) + (y >= 0.75) + (y > 1.25) + (y >= 1.75) + (y > 2.5) + (y >= 3.5) + (y > 5.0))
    code = (code + 8 * (torch.signbit(x) & fine[..., None])).to(torch.uint8).flatten(-2)
    code = code[..., 0::2] + 16 * code[..., 1::2]
    scale = torch.where(fine, s.half().view(torch.int16) >> 7, 0xFC).to(torch.uint8)
    rows = torch.cat([code, scale], -1)
    return torch.nn.functional.pad(rows, (0, row_bytes(d) - rows.shape[-1]))


def unpack(rows, d):
    """The values of such rows in float32, [..., d]."""
    g = -(-d // 16)
    table = torch.tensor(VALUES + tuple(-v for v in VALUES), device=rows.device)
    code = rows[..., :8 * g]
    x = table[torch.stack([code & 15, code >> 4], -1).int()].flatten(-2)
    s = (rows[..., 8 * g:9 * g].to(torch.int16) << 7).view(torch.float16).float()
    return (x.reshape(*x.shape[:-1], g, 16) * s[..., None]).flatten(-2)[..., :d]


# ---- inputs ------------------------------------------------------------------

def parents_of(c):
    p = [[i // c["branch"] - 1 if i < m else -2 for i in range(c["nodes"])] for m in nodes_of(c)]
    return torch.tensor(p, dtype=torch.int32, device=DEVICE)


def prepare(c, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    t, b, op, hk, d = DTYPES[c["dtype"]], c["batch"], c["op"], c["kv_heads"], c["head_dim"]
    normal = lambda *s: torch.randn(*s, generator=g, device=DEVICE, dtype=torch.float32)  # noqa: E731
    # elements of a head differ in size, as trained keys' do
    size = torch.exp(0.5 * normal(hk, d))
    s = {"case": c, "cc": context() if own else None}
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEVICE)  # noqa: E731
    if op in ("prompt", "fill"):
        starts = [0]
        for n in lengths(c):
            starts.append(starts[-1] + n)
        rows = starts[-1] + c.get("spare", 0)
        s["starts"] = i32(starts)
        s["k"], s["v"] = (size * normal(rows, hk, d)).to(t), normal(rows, hk, d).to(t)
        if op == "prompt":
            # queries that look for some of the keys, as trained heads do
            s["q"] = (1.5 * normal(rows, c["q_heads"], d)).to(t)
            return s
        s["lens"] = i32([c["cached"]] * b)
    else:
        s["lens"] = i32(lengths(c))
    cap = capacity(c)
    s["k_cache"] = pack(size[:, None] * normal(b, hk, cap, d))
    s["v_cache"] = pack(normal(b, hk, cap, d))
    if op == "fill":
        return s
    n = c["nodes"]
    s["k_new"], s["v_new"] = (size * normal(b, n, hk, d)).to(t), normal(b, n, hk, d).to(t)
    if op == "attend":
        s["q"] = (1.5 * normal(b, n, c["q_heads"], d)).to(t)
        return s | {"parents": parents_of(c)}
    path = path_of(c)
    s["path"] = i32([path + [-1] * (n - len(path))] * b)
    s["count"] = i32(counts(c))
    return s


# ---- the plain forms -----------------------------------------------------------

def softmax_rows(x, values):
    """Weights, sums and their logs of the scores x [..., rows, keys] over values [..., keys, d]; a row without a key
    is 0, its log -inf."""
    top = x.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), 0.0, top)
    p = torch.exp(x - top)
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, values) / torch.where(total > 0, total, 1.0)
    return out, (torch.log(total) + top)[..., 0]


def plain_prompt(s):
    q, k, v, starts, c = s["q"], s["k"], s["v"], s["starts"].long(), s["case"]
    t, hq, d = q.shape
    hk, n, b = k.shape[1], max(lengths(c)), c["batch"]
    at = torch.arange(n, device=q.device)
    real = at < (starts[1:] - starts[:-1])[:, None]  # [b, n]
    row = torch.where(real, starts[:-1, None] + at, 0)
    take = lambda x: x[row].float().transpose(1, 2)  # noqa: E731
    keys, values = take(k), torch.where(real[:, None, :, None], take(v), 0.0)
    x = torch.matmul(take(q).reshape(b, hk, hq // hk, n, d), keys[:, :, None].transpose(3, 4)) / math.sqrt(d)
    sees = real[:, None, :] & (at <= at[:, None])
    x = torch.where(sees[:, None, None], x, -math.inf)
    y, log = softmax_rows(x, values[:, :, None])
    out = torch.zeros(t + 1, hq, d, device=q.device)
    lse = torch.full((t + 1, hq), -math.inf, device=q.device)
    row = torch.where(real, row, t)  # what belongs to no sequence goes behind the rest
    out[row] = y.reshape(b, hq, n, d).transpose(1, 2)
    lse[row] = log.reshape(b, hq, n).transpose(1, 2)
    return out[:t].to(q.dtype), lse[:t]


def read_back(s, lens):
    d, t = s["case"]["head_dim"], DTYPES[s["case"]["dtype"]]
    held = torch.arange(s["k_cache"].shape[2], device=lens.device) < lens[:, None]
    return tuple(torch.where(held[:, None, :, None], unpack(s[x], d), 0.0).to(t) for x in ("k_cache", "v_cache"))


def plain_fill(s):
    lens, starts = s["lens"], s["starts"]
    t = torch.arange(s["k"].shape[0], device=lens.device, dtype=torch.int32)
    b = torch.searchsorted(starts, t, right=True) - 1  # the sequence of each row
    slot = (lens[b] + t - starts[b]).long()
    s["k_cache"][b, :, slot], s["v_cache"][b, :, slot] = pack(s["k"]), pack(s["v"])
    lens = lens + starts[1:] - starts[:-1]
    return *read_back(s, lens), lens


def plain_commit(s):
    lens, path, count = s["lens"], s["path"], s["count"]
    n = path.shape[1]
    j, each = torch.arange(n, device=lens.device), torch.arange(path.shape[0], device=lens.device)[:, None]
    slot, node = (lens[:, None] + j).long(), path.clamp(min=0).long()
    real = (j < count[:, None])[..., None, None]
    for cache, fresh in ((s["k_cache"], s["k_new"]), (s["v_cache"], s["v_new"])):
        cache[each, :, slot] = torch.where(real, pack(fresh[each, node]), cache[each, :, slot])
    return *read_back(s, lens + count), lens + count


def reach(parents):
    """[b, i, j]: j is i or an ancestor of i; and whether node i belongs to the tree."""
    n = parents.shape[1]
    at = torch.arange(n, device=parents.device)
    up = (parents[..., None] == at) & (at < at[:, None])
    # entries of (1 + up)^n are positive exactly where a walk upwards leads
    r = torch.linalg.matrix_power(up.double() + torch.eye(n, device=parents.device, dtype=torch.float64), n) > 0
    inside = (r & (parents == -1)[:, None]).any(-1)
    return r & inside[..., None]


def plain_attend(s):
    q, kn, vn = (s[x].float() for x in ("q", "k_new", "v_new"))
    b, n, hq, d = q.shape
    hk, cap = s["k_cache"].shape[1:3]
    q = q.reshape(b, n, hk, hq // hk, d).permute(0, 2, 3, 1, 4).reshape(b, hk, -1, d)
    sees = reach(s["parents"])
    inside = sees.diagonal(dim1=1, dim2=2)
    held = torch.arange(cap, device=q.device) < s["lens"][:, None]
    mask = torch.cat([held[:, None] & inside[..., None], sees], -1)  # [b, n, cap + n]
    mask = mask[:, None, None].expand(b, 1, hq // hk, n, cap + n).reshape(b, 1, -1, cap + n)
    keys = torch.cat([unpack(s["k_cache"], d), kn.transpose(1, 2)], 2)
    usable = torch.cat([held, inside], -1)[:, None, :, None]
    values = torch.where(usable, torch.cat([unpack(s["v_cache"], d), vn.transpose(1, 2)], 2), 0.0)
    x = torch.where(mask, torch.matmul(q, keys.transpose(2, 3)) / math.sqrt(d), -math.inf)
    out, lse = softmax_rows(x, values)
    back = lambda y: y.reshape(b, hk, hq // hk, n, -1).permute(0, 3, 1, 2, 4).reshape(b, n, hq, -1)  # noqa: E731
    return back(out).to(s["q"].dtype).contiguous(), back(lse[..., None])[..., 0].contiguous()


PLAIN = {"prompt": plain_prompt, "fill": plain_fill, "commit": plain_commit, "attend": plain_attend}


def run(s):
    op = s["case"]["op"]
    if not own:
        return PLAIN[op](s)
    cc, d, t = s["cc"], s["case"]["head_dim"], DTYPES[s["case"]["dtype"]]
    if op == "prompt":
        return cc.draft_prompt(s["q"], s["k"], s["v"], s["starts"])
    if op == "attend":
        return cc.draft_attention4(s["q"], s["k_cache"], s["v_cache"], s["lens"], s["k_new"], s["v_new"], s["parents"])
    if op == "fill":
        lens = cc.draft_fill4(s["k_cache"], s["v_cache"], s["lens"], s["k"], s["v"], s["starts"])
    else:
        lens = cc.draft_commit4(s["k_cache"], s["v_cache"], s["lens"], s["k_new"], s["v_new"], s["path"], s["count"])
    return cc.draft_read4(s["k_cache"], lens, d, t), cc.draft_read4(s["v_cache"], lens, d, t), lens


# ---- the definitions in 64 bits -----------------------------------------------

def values_of(rows, d):
    """The values of 4-bit rows, from the bits: (-1)^s 2^(e - 1) (1 + m / 2), or s m / 2 where e = 0."""
    g = -(-d // 16)
    code = torch.stack([rows[..., :8 * g] % 16, rows[..., :8 * g] // 16], -1).flatten(-2).double()
    sign, e, m = torch.floor(code / 8), torch.floor(code / 2) % 4, code % 2
    x = (1 - 2 * sign) * torch.where(e > 0, torch.exp2(e - 1) * (1 + m / 2), m / 2)
    b = rows[..., 8 * g:9 * g].double()
    e, m = torch.floor(b / 8), b % 8
    s = torch.where(e > 0, torch.exp2(e - 15) * (1 + m / 8), torch.exp2(torch.full_like(m, -14.0)) * m / 8)
    s = torch.where(e == 31, math.nan, s)
    return (x * s.repeat_interleave(16, -1))[..., :d]


def nearest(x, table):
    """The index of the nearest of the rising values, the even one in the middle."""
    hi = torch.searchsorted(table, x).clamp(1, len(table) - 1)
    lo = hi - 1
    a, b = x - table[lo], table[hi] - x
    return torch.where((b < a) | ((a == b) & (hi % 2 == 0)), hi, lo)


def quantised(x):
    """What x [..., d] becomes in a 4-bit cache, in 64 bits (finite values)."""
    d = x.shape[-1]
    pad = x.new_zeros(*x.shape[:-1], -d % 16).double()
    x = torch.cat([x.double(), pad], -1)
    x = x.unflatten(-1, (-(-d // 16), 16))
    scales = [m / 8 * 2.0 ** -14 for m in range(8)]
    scales += [(1 + m / 8) * 2.0 ** e for e in range(-14, 14) for m in range(8) if (1 + m / 8) * 2.0 ** e <= TOP]
    scales = torch.tensor(scales, dtype=torch.float64, device=x.device)
    s = scales[nearest(x.abs().amax(-1) / 6, scales)][..., None]
    few = torch.tensor(VALUES, dtype=torch.float64, device=x.device)
    y = few[nearest(x.abs() / torch.where(s > 0, s, 1.0), few)] * s * torch.sign(x)
    return y.flatten(-2)[..., :d]


def exact_prompt(s):
    q, starts = s["q"], s["starts"].tolist()
    t, hq, d = q.shape
    hk = s["k"].shape[1]
    out = torch.zeros(t, hq, d, dtype=torch.float64, device=q.device)
    lse = torch.full((t, hq), -math.inf, dtype=torch.float64, device=q.device)
    for a, e in zip(starts, starts[1:]):
        later = torch.ones(e - a, e - a, dtype=torch.bool, device=q.device).triu(1)
        for h in range(hq):
            k, v = (s[x][a:e, h // (hq // hk)].double() for x in ("k", "v"))
            z = (q[a:e, h].double() @ k.T * d ** -0.5).masked_fill(later, -math.inf)
            lse[a:e, h] = torch.logsumexp(z, 1)
            out[a:e, h] = torch.exp(z - lse[a:e, h][:, None]) @ v
    return out, lse


def exact_read(s, lens, rows):
    """The caches' values with rows (sequence, slot, key rows, value rows) written."""
    d = s["case"]["head_dim"]
    got = []
    for x, at in (("k_cache", 2), ("v_cache", 3)):
        y = values_of(s[x], d)
        for r in rows:
            y[r[0], :, r[1]] = quantised(r[at]).movedim(0, y[r[0], :, r[1]].dim() - 2)
        for i, m in enumerate(lens.tolist()):
            y[i, :, m:] = 0.0
        got.append(y)
    return *got, lens


def exact_fill(s):
    starts, lens = s["starts"].tolist(), s["lens"].clone()
    rows = []
    for i, (a, e) in enumerate(zip(starts, starts[1:])):
        m = int(lens[i])
        rows.append((i, slice(m, m + e - a), s["k"][a:e], s["v"][a:e]))
        lens[i] += e - a
    return exact_read(s, lens, rows)


def exact_commit(s):
    lens, rows = s["lens"].clone(), []
    for i, (m, a) in enumerate(zip(s["lens"].tolist(), s["count"].tolist())):
        path = s["path"][i, :a].long()
        rows.append((i, slice(m, m + a), s["k_new"][i, path], s["v_new"][i, path]))
        lens[i] += a
    return exact_read(s, lens, rows)


def ancestors(parents, i):
    """The nodes that node i of one tree sees, or none where it is not of the tree."""
    got = []
    while 0 <= i < len(parents):
        got.append(i)
        if parents[i] >= i:
            return []
        i = parents[i]
    return sorted(got) if i == -1 else []


def exact_attend(s):
    q, b = s["q"], s["q"].shape[0]
    n, hq, d = q.shape[1:]
    hk = s["k_cache"].shape[1]
    out = torch.zeros(b, n, hq, d, dtype=torch.float64, device=q.device)
    lse = torch.full((b, n, hq), -math.inf, dtype=torch.float64, device=q.device)
    for i, (m, tree) in enumerate(zip(s["lens"].tolist(), s["parents"].tolist())):
        see = [ancestors(tree, j) for j in range(n)]
        rows = [j for j in range(n) if see[j]]
        hide = torch.ones(len(rows), n, dtype=torch.bool, device=q.device)
        for r, j in enumerate(rows):
            hide[r, see[j]] = False
        spare = torch.tensor([not see[j] for j in range(n)], device=q.device)
        for h in range(hk):
            k, v = values_of(s["k_cache"][i, h, :m], d), values_of(s["v_cache"][i, h, :m], d)
            kn = s["k_new"][i, :, h].double().masked_fill(spare[:, None], 0.0)
            vn = s["v_new"][i, :, h].double().masked_fill(spare[:, None], 0.0)
            for x in range(h * (hq // hk), (h + 1) * (hq // hk)):
                y = q[i, rows, x].double() * d ** -0.5
                z = torch.cat([y @ k.T, (y @ kn.T).masked_fill(hide, -math.inf)], 1)
                lse[i, rows, x] = torch.logsumexp(z, 1)
                z = torch.exp(z - lse[i, rows, x][:, None])
                out[i, rows, x] = z[:, :m] @ v + z[:, m:] @ vn
    return out, lse


EXACT = {"prompt": exact_prompt, "fill": exact_fill, "commit": exact_commit, "attend": exact_attend}


def exact(c, seed):
    return EXACT[c["op"]](prepare(c, seed))
