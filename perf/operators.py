"""The drafted-decoding operators of the data owner, as measured cases.

An encrypted forward costs about the same for one token as for a few dozen
(32 tokens share a ciphertext), so the data owner drafts several tokens with a
small plain model of its own, has the encrypted model evaluate all of them in
one forward, and keeps the ones that the encrypted model's probabilities
confirm.  The operators are what that owner runs in plain on its GPU:

  attend      attention of a tree of drafted tokens over the draft model's
              key/value cache (one node is the single-token decode step)
  verify      acceptance of the drafts against the target's probabilities from
              given random numbers, and the token that follows them
  commit      the accepted nodes' keys and values appended to the cache
  accumulate  the attention weight that the accepted nodes give each cached key
  evict       the cache cut to a budget: the latest keys and the heaviest ones

``run`` is the plain form in torch when ``own`` is false, and the calls of this
repository's ``CryptoContext`` when it is true.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "fp64": torch.float64}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4, "fp64": 8}
DEVICE = "cuda"

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
        # the draft model's next token behind a prompt of 103 tokens: 12 heads of 64, one node; latency
        dict(name="attend one node, 103 keys", op="attend", dtype="bf16", batch=1, nodes=1, branch=1, q_heads=12,
             kv_heads=12, head_dim=64, length=103, ragged=False),
        # eight sequences, each a binary tree of 21 drafts over a context of some thousand tokens, padded batch
        dict(name="attend trees of 21, 4001 keys", op="attend", dtype="fp16", batch=8, nodes=21, branch=2, q_heads=12,
             kv_heads=12, head_dim=64, length=4001, ragged=True),
        # a long genomic context and a draft model with shared key/value heads: 4 query heads on each
        dict(name="attend trees of 32, 65536 keys", op="attend", dtype="bf16", batch=2, nodes=32, branch=3, q_heads=32,
             kv_heads=8, head_dim=128, length=65536, ragged=False),
        # a draft model kept in 32 bits
        dict(name="attend chains of 5, fp32", op="attend", dtype="fp32", batch=4, nodes=5, branch=1, q_heads=12,
             kv_heads=12, head_dim=64, length=6000, ragged=True),
        # one sequence, five drafts in a row, probabilities of the decrypted model in 64 bits, 6-mers as tokens
        dict(name="verify a chain of 5, fp64", op="verify", dtype="fp64", batch=1, nodes=5, branch=1, vocab=4103),
        # a served batch of trees over a large vocabulary
        dict(name="verify trees of 31", op="verify", dtype="fp32", batch=64, nodes=31, branch=2, vocab=32003),
        # one layer's cache after a chain of drafts
        dict(name="commit a chain", op="commit", dtype="bf16", batch=1, nodes=5, branch=1, kv_heads=12, head_dim=64,
             length=1000, accepted=3),
        # a served batch, wide trees
        dict(name="commit from trees", op="commit", dtype="fp32", batch=32, nodes=64, branch=2, kv_heads=16,
             head_dim=128, length=2000, accepted=6),
        # the weights of a few accepted nodes over an ordinary context
        dict(name="accumulate over 4001 keys", op="accumulate", dtype="fp16", batch=8, nodes=21, branch=2, q_heads=12,
             kv_heads=12, head_dim=64, length=4001, accepted=4),
        # and over a long one, four query heads on each key
        dict(name="accumulate over 65536 keys", op="accumulate", dtype="bf16", batch=2, nodes=32, branch=3, q_heads=32,
             kv_heads=8, head_dim=128, length=65536, accepted=4),
        # an ordinary cache cut to half
        dict(name="evict 2100 to 1000", op="evict", dtype="bf16", batch=1, kv_heads=12, head_dim=64, length=2100,
             budget=1000, recent=100),
        # a long prompt cut to the budget that decoding keeps
        dict(name="evict 65536 to 16384", op="evict", dtype="bf16", batch=4, kv_heads=8, head_dim=128, length=65536,
             budget=16384, recent=1024),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "verify", "commit", "accumulate", "evict"])
    if op == "verify":
        return dict(op=op, dtype=rng.choice(["fp32", "fp64"]), batch=_log(rng, 1, 48), nodes=rng.randint(1, 31),
                    branch=rng.randint(1, 4), vocab=_log(rng, 16, 32000))
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    kv_heads, head_dim = rng.choice([1, 2, 4, 8, 12, 16]), rng.choice([32, 64, 64, 80, 96, 128])
    c = dict(op=op, dtype=dtype, batch=_log(rng, 1, 16), kv_heads=kv_heads, head_dim=head_dim, length=1)
    # at most 2^26 values in the keys (the largest listed cache holds four times that)
    c["length"] = _log(rng, 1, max(2, min(65536, (1 << 26) // (c["batch"] * kv_heads * head_dim))))
    if op == "evict":
        c["budget"] = rng.randint(1, max(1, c["length"]))
        c["recent"] = rng.randint(0, c["budget"])
        return c
    c["nodes"], c["branch"] = _log(rng, 1, 64), rng.randint(1, 4)
    if op != "commit":
        c["q_heads"] = kv_heads * rng.choice([1, 1, 2, 4] if c["nodes"] <= 32 else [1, 1, 2])
    if op == "attend":
        c["ragged"] = rng.random() < 0.5
    else:
        c["accepted"] = rng.randint(1, 8)
    return c


def lengths(c):
    """Cached keys of each sequence: the whole length down to half of it, none in the last of a large batch."""
    n, b = c["length"], c["batch"]
    got = [n - (n // 2) * i // b for i in range(b)]
    if b >= 6:
        got[-1] = 0
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


def work(c):
    e, b, op = BYTES[c["dtype"]], c["batch"], c["op"]
    if op == "verify":
        # one row of the target and one of the draft decide a sequence's next token
        return {"bytes": b * (2 * c["vocab"] * e + c["nodes"] * (16 + 2 * e) + 16), "flops": 3 * b * c["vocab"]}
    hk, d = c["kv_heads"], c["head_dim"]
    keys = sum(lengths(c))
    if op == "attend":
        hq, n = c["q_heads"], c["nodes"]
        seen = sum(m * s + depth_sum(c, m) for m, s in zip(nodes_of(c), lengths(c)))
        return {"bytes": e * d * (2 * hk * (keys + sum(nodes_of(c))) + 2 * b * n * hq) + 4 * b * n * hq,
                "flops": 4 * hq * d * seen}
    if op == "commit":
        return {"bytes": 4 * e * hk * d * sum(counts(c)) + 16 * b, "flops": 0}
    if op == "accumulate":
        keys = sum(m + a for m, a in zip(lengths(c), counts(c)) if a)
        return {"bytes": hk * keys * (e * d + 8) + sum(counts(c)) * c["q_heads"] * (e * d + 4) + 8 * b,
                "flops": 2 * c["q_heads"] * d * sum(a * m for m, a in zip(lengths(c), counts(c)))}
    kept = sum(min(s, c["budget"]) for s in lengths(c))
    return {"bytes": hk * (4 * keys + kept * (4 * d * e + 8)), "flops": 0}


# ---- inputs ------------------------------------------------------------------

def parents_of(c):
    p = [[i // c["branch"] - 1 if i < m else -2 for i in range(c["nodes"])] for m in nodes_of(c)]
    return torch.tensor(p, dtype=torch.int32, device=DEVICE)


def prepare(c, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    t, b, op = DTYPES[c["dtype"]], c["batch"], c["op"]
    normal = lambda *s: torch.randn(*s, generator=g, device=DEVICE, dtype=torch.float32)  # noqa: E731
    s = {"case": c, "cc": context() if own else None}
    if op == "verify":
        n, v = c["nodes"], c["vocab"]
        logits = 2.5 * normal(b, n + 1, v)
        target = torch.softmax(logits.to(t), -1)
        draft = torch.softmax((logits + 0.7 * normal(b, n + 1, v)).to(t), -1)
        parents = parents_of(c)
        rows = draft.gather(1, (parents + 1).long()[..., None].expand(b, n, v)).reshape(b * n, v)
        tokens = torch.multinomial(rows, 1, generator=g).reshape(b, n).to(torch.int32)
        uniforms = torch.rand(b, n + 1, generator=g, device=DEVICE, dtype=torch.float64)
        return s | {"target": target, "draft": draft, "tokens": tokens, "parents": parents, "uniforms": uniforms}
    hk, d = c["kv_heads"], c["head_dim"]
    cap = c["length"] + c.get("nodes", 0)
    s["lens"] = torch.tensor(lengths(c), dtype=torch.int32, device=DEVICE)
    s["k_cache"], s["v_cache"] = normal(b, hk, cap, d).to(t), normal(b, hk, cap, d).to(t)
    if op == "evict":
        # weights as sums of softmax rows leave them: most keys light, some heavy
        s["acc"] = torch.exp(2.0 * normal(b, hk, cap))
        s["out"] = (torch.zeros(b, hk, c["budget"], d, dtype=t, device=DEVICE),
                    torch.zeros(b, hk, c["budget"], d, dtype=t, device=DEVICE),
                    torch.zeros(b, hk, c["budget"], device=DEVICE))
        return s
    n = c["nodes"]
    if op in ("attend", "accumulate"):
        hq = c["q_heads"]
        # queries that look for some of the keys, as trained heads do
        s["q"] = (1.5 * normal(b, n, hq, d)).to(t)
    if op in ("attend", "commit"):
        s["k_new"], s["v_new"] = normal(b, n, hk, d).to(t), normal(b, n, hk, d).to(t)
    if op == "attend":
        return s | {"parents": parents_of(c)}
    path = path_of(c)
    s["path"] = torch.tensor([path + [-1] * (n - len(path))] * b, dtype=torch.int32, device=DEVICE)
    s["count"] = torch.tensor(counts(c), dtype=torch.int32, device=DEVICE)
    if op == "accumulate":
        s["acc"] = torch.rand(b, hk, cap, generator=g, device=DEVICE)
        # the log of each row's sum, as attention over the same keys returned it
        s["lse"] = torch.zeros(b, n, hq, device=DEVICE)
        if path:
            rows = s["q"][:, path].float().reshape(b, len(path), hk, hq // hk, d)
            for i, m in enumerate(lengths(c)):
                keys = s["k_cache"][i, :, :m + len(path)].float()
                x = torch.einsum("jhgd,hsd->jhgs", rows[i], keys) / math.sqrt(d)
                later = torch.arange(m + len(path), device=DEVICE) > m + torch.arange(len(path), device=DEVICE)[:, None]
                x = x.masked_fill(later[:, None, None], -math.inf)
                s["lse"][i, path] = torch.logsumexp(x, -1).reshape(len(path), hq)
    return s


# ---- the plain forms -----------------------------------------------------------

def reach(parents):
    """[b, i, j]: j is i or an ancestor of i; and whether node i belongs to the tree."""
    n = parents.shape[1]
    at = torch.arange(n, device=parents.device)
    up = (parents[..., None] == at) & (at < at[:, None])
    # entries of (1 + up)^n are positive exactly where a walk upwards leads
    r = torch.linalg.matrix_power(up.double() + torch.eye(n, device=parents.device, dtype=torch.float64), n) > 0
    inside = (r & (parents == -1)[:, None]).any(-1)
    return r & inside[..., None], inside


def plain_attend(s):
    q, k, v, kn, vn = (s[x].float() for x in ("q", "k_cache", "v_cache", "k_new", "v_new"))
    b, n, hq, d = q.shape
    hk, cap = k.shape[1:3]
    q = q.reshape(b, n, hk, hq // hk, d).permute(0, 2, 3, 1, 4).reshape(b, hk, -1, d)
    sees, _ = reach(s["parents"])
    held = (torch.arange(cap, device=q.device) < s["lens"][:, None])
    inside = sees.diagonal(dim1=1, dim2=2)
    mask = torch.cat([held[:, None] & inside[..., None], sees], -1)  # [b, n, cap + n]
    mask = mask[:, None, None].expand(b, 1, hq // hk, n, cap + n).reshape(b, 1, -1, cap + n)
    keys = torch.cat([k, kn.transpose(1, 2)], 2)
    usable = torch.cat([held, inside], -1)[:, None, :, None]
    values = torch.where(usable, torch.cat([v, vn.transpose(1, 2)], 2), 0.0)
    x = torch.where(mask, torch.matmul(q, keys.transpose(2, 3)) / math.sqrt(d), -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(torch.isinf(top), 0.0, top))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, values) / torch.where(total > 0, total, 1.0)
    lse = (torch.log(total) + torch.where(total > 0, top, 0.0))[..., 0]
    back = lambda y: y.reshape(b, hk, hq // hk, n, -1).permute(0, 3, 1, 2, 4).reshape(b, n, hq, -1)  # noqa: E731
    return back(out).to(s["q"].dtype).contiguous(), back(lse)[..., 0].contiguous()


def plain_verify(s):
    target, draft, tokens, parents, u = (s[x] for x in ("target", "draft", "tokens", "parents", "uniforms"))
    b, n = tokens.shape
    v = target.shape[2]
    each = torch.arange(b, device=tokens.device)
    at = torch.full((b,), -1, dtype=torch.int32, device=tokens.device)  # the node reached so far
    count = torch.zeros_like(at)
    path = torch.full((b, n + 1), -1, dtype=torch.int32, device=tokens.device)
    p, q = target[:, 0].double(), draft[:, 0].double()
    for i in range(n):  # a node comes behind its parent and its earlier siblings
        x = tokens[:, i].long()
        known = (x >= 0) & (x < v)
        px, qx = (y.gather(1, x.clamp(0, v - 1)[:, None])[:, 0] for y in (p, q))
        asked = parents[:, i] == at
        yes = asked & known & (u[:, i] * qx < px)
        rest = torch.clamp(p - q, min=0.0)
        mass = rest.sum(-1, keepdim=True)
        p = torch.where((asked & ~yes)[:, None] & (mass > 0), rest / torch.where(mass > 0, mass, 1.0), p)
        p = torch.where(yes[:, None], target[:, i + 1].double(), p)
        q = torch.where(yes[:, None], draft[:, i + 1].double(), q)
        slot = torch.where(yes, count, n).long()
        path[each, slot] = i
        at = torch.where(yes, i, at)
        count = count + yes
    path[:, n] = -1
    cdf = torch.cumsum(p, -1)
    over = cdf > u[:, n:] * p.sum(-1, keepdim=True)
    last = torch.where(p > 0, torch.arange(v, device=p.device), 0).amax(-1)
    token = torch.where(over.any(-1), over.to(torch.uint8).argmax(-1), last)
    return path[:, :n].contiguous(), count.to(torch.int32), token.to(torch.int32)


def plain_commit(s):
    k, v, kn, vn, lens, path, count = (s[x] for x in ("k_cache", "v_cache", "k_new", "v_new", "lens", "path", "count"))
    n = path.shape[1]
    j, each = torch.arange(n, device=k.device), torch.arange(k.shape[0], device=k.device)[:, None]
    slot, node = (lens[:, None] + j).long(), path.clamp(min=0).long()
    real = (j < count[:, None])[..., None, None]
    for cache, fresh in ((k, kn), (v, vn)):
        cache[each, :, slot] = torch.where(real, fresh[each, node], cache[each, :, slot])
    return k, v, lens + count


def plain_accumulate(s):
    q, k, lse, lens, path, count, acc = (s[x] for x in ("q", "k_cache", "lse", "lens", "path", "count", "acc"))
    b, n, hq, d = q.shape
    hk, cap = k.shape[1:3]
    most = max(1, len(path_of(s["case"])))
    node = path[:, :most].clamp(min=0).long()
    rows = q.float().gather(1, node[..., None, None].expand(b, most, hq, d))
    rows = rows.reshape(b, most, hk, hq // hk, d).permute(0, 2, 1, 3, 4).reshape(b, hk, -1, d)
    tops = lse.gather(1, node[..., None].expand(b, most, hq))
    tops = tops.reshape(b, most, hk, hq // hk).permute(0, 2, 1, 3).reshape(b, hk, -1, 1)
    x = torch.matmul(rows, k.float().transpose(2, 3)) / math.sqrt(d) - tops
    at, j = torch.arange(cap, device=k.device), torch.arange(most, device=k.device)
    sees = (at <= lens[:, None, None] + j[:, None]) & (j < count[:, None])[..., None]  # [b, most, cap]
    sees = sees[:, None, :, None].expand(b, 1, most, hq // hk, cap).reshape(b, 1, -1, cap)
    more = torch.where(sees, torch.exp(torch.where(sees, x, 0.0)), 0.0).sum(2)
    old, held = at < lens[:, None], at < (lens + count)[:, None]
    acc.copy_(torch.where(held[:, None], torch.where(old[:, None], acc, 0.0) + more, acc))
    return acc


def plain_evict(s):
    k, v, acc, lens, (k2, v2, acc2) = s["k_cache"], s["v_cache"], s["acc"], s["lens"], s["out"]
    b, hk, cap, d = k.shape
    budget, recent = s["case"]["budget"], s["case"]["recent"]
    at = torch.arange(cap, device=k.device)
    held = (at < lens[:, None])[:, None].expand(b, hk, cap)
    latest = held & (at >= lens[:, None] - recent)[:, None]
    # the latest keys first, then the heaviest, the lower index first among equals, then what is not held
    first = torch.where(latest, math.inf, torch.where(held, acc.double(), -math.inf))
    order = torch.sort(first, dim=-1, descending=True, stable=True).indices
    chosen = order[..., :budget]
    chosen = torch.where(held.gather(2, chosen), chosen, cap)  # what is not held goes behind
    chosen = torch.sort(chosen, dim=-1).values
    real = chosen < cap
    take = chosen.clamp(max=cap - 1)
    rows = take[..., None].expand(b, hk, budget, d)
    k2.copy_(torch.where(real[..., None], k.gather(2, rows), k2))
    v2.copy_(torch.where(real[..., None], v.gather(2, rows), v2))
    acc2.copy_(torch.where(real, acc.gather(2, take), acc2))
    return k2, v2, acc2, torch.where(real, take, -1).to(torch.int32), lens.clamp(max=budget)


PLAIN = {"attend": plain_attend, "verify": plain_verify, "commit": plain_commit, "accumulate": plain_accumulate,
         "evict": plain_evict}


def run(s):
    op = s["case"]["op"]
    if not own:
        return PLAIN[op](s)
    cc = s["cc"]
    if op == "attend":
        return cc.draft_attention(s["q"], s["k_cache"], s["v_cache"], s["lens"], s["k_new"], s["v_new"], s["parents"])
    if op == "verify":
        return cc.draft_verify(s["target"], s["draft"], s["tokens"], s["parents"], s["uniforms"])
    if op == "commit":
        lens = cc.draft_commit(s["k_cache"], s["v_cache"], s["lens"], s["k_new"], s["v_new"], s["path"], s["count"])
        return s["k_cache"], s["v_cache"], lens
    if op == "accumulate":
        return cc.draft_accumulate(s["q"], s["lse"], s["k_cache"], s["lens"], s["path"], s["count"], s["acc"])
    return cc.draft_evict(s["k_cache"], s["v_cache"], s["acc"], s["lens"], s["case"]["budget"], s["case"]["recent"],
                          out=s["out"])


# ---- the definitions in 64 bits -----------------------------------------------

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
            k, v = s["k_cache"][i, h, :m].double(), s["v_cache"][i, h, :m].double()
            kn = s["k_new"][i, :, h].double().masked_fill(spare[:, None], 0.0)
            vn = s["v_new"][i, :, h].double().masked_fill(spare[:, None], 0.0)
            for x in range(h * (hq // hk), (h + 1) * (hq // hk)):
                y = q[i, rows, x].double() * d ** -0.5
                z = torch.cat([y @ k.T, (y @ kn.T).masked_fill(hide, -math.inf)], 1)
                lse[i, rows, x] = torch.logsumexp(z, 1)
                z = torch.exp(z - lse[i, rows, x][:, None])
                out[i, rows, x] = z[:, :m] @ v + z[:, m:] @ vn
    return out, lse


def exact_verify(s):
    b, n = s["tokens"].shape
    paths, counts, picks = [], [], []
    for i in range(b):
        tokens, tree, u = s["tokens"][i].tolist(), s["parents"][i].tolist(), s["uniforms"][i].tolist()
        path, node, go = [], -1, True
        while go:
            p, q, go = s["target"][i, node + 1].double(), s["draft"][i, node + 1].double(), False
            for j in [j for j in range(n) if tree[j] == node and j > node]:
                if 0 <= tokens[j] < p.numel() and u[j] * q[tokens[j]].item() < p[tokens[j]].item():
                    path.append(j)
                    node, go = j, True
                    break
                rest = (p - q).clamp(min=0.0)
                if rest.sum().item() > 0:
                    p = rest / rest.sum()
        cdf = p.cumsum(0)
        hit = (cdf > u[n] * cdf[-1]).nonzero()
        picks.append(int(hit[0] if len(hit) else p.nonzero()[-1]))
        counts.append(len(path))
        paths.append(path + [-1] * (n - len(path)))
    return tuple(torch.tensor(x, dtype=torch.int32) for x in (paths, counts, picks))


def exact_commit(s):
    k, v, lens = s["k_cache"].double(), s["v_cache"].double(), s["lens"].clone()
    for i, (m, a) in enumerate(zip(s["lens"].tolist(), s["count"].tolist())):
        for j in range(a):
            node = int(s["path"][i, j])
            k[i, :, m + j], v[i, :, m + j] = s["k_new"][i, node].double(), s["v_new"][i, node].double()
        lens[i] += a
    return k, v, lens


def exact_accumulate(s):
    acc = s["acc"].double()
    hq, d = s["q"].shape[2:]
    hk = acc.shape[1]
    for i, (m, a) in enumerate(zip(s["lens"].tolist(), s["count"].tolist())):
        acc[i, :, m:m + a] = 0.0
        for j in range(a):
            node = int(s["path"][i, j])
            for x in range(hq):
                h = x // (hq // hk)
                z = s["k_cache"][i, h, :m + j + 1].double() @ s["q"][i, node, x].double() * d ** -0.5
                acc[i, h, :m + j + 1] += torch.exp(z - s["lse"][i, node, x].double())
    return acc


def exact_evict(s):
    k2, v2, acc2 = (x.double() for x in s["out"])
    b, hk = s["acc"].shape[:2]
    budget, recent = s["case"]["budget"], s["case"]["recent"]
    index = torch.full((b, hk, budget), -1, dtype=torch.int32, device=k2.device)
    for i, m in enumerate(s["lens"].tolist()):
        for h in range(hk):
            keep = torch.arange(m, device=k2.device)
            if m > budget:
                w = s["acc"][i, h, :m - recent].cpu().numpy()
                heavy = (-w.astype("f8")).argsort(kind="stable")[:budget - recent]
                keep = torch.cat([torch.from_numpy(heavy).to(k2.device).sort().values, keep[m - recent:]])
            a = keep.numel()
            k2[i, h, :a], v2[i, h, :a] = s["k_cache"][i, h, keep].double(), s["v_cache"][i, h, keep].double()
            acc2[i, h, :a] = s["acc"][i, h, keep].double()
            index[i, h, :a] = keep.int()
    return k2, v2, acc2, index, torch.clamp(s["lens"], max=budget)


EXACT = {"attend": exact_attend, "verify": exact_verify, "commit": exact_commit, "accumulate": exact_accumulate,
         "evict": exact_evict}


def exact(c, seed):
    return EXACT[c["op"]](prepare(c, seed))
