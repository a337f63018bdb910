"""The operators of a step that checks drafted tokens, as cases that can be timed and compared.

Several tokens of a request are drafted ahead, as a tree (a row per token; row 0 is the request's last known token, every
other row names its parent among the rows before it).  One step runs all rows:

    layout    the step's tables built on the device from the requests' lengths: span starts, positions, the pages' slots,
              block tables, and which rows of its own span a row sees (its ancestors and itself)
    tree      attention of the rows over their requests' cached keys and the drafted rows that they see
    logprobs  log probabilities of given tokens with the rows' entropy, the tokens' ranks and the best alternatives
    accept    the walk down each tree along the tokens that the model chose itself
    commit    keys and values of the accepted rows written into the cache, all layers at once

A case's `rows` and `contexts` say what the requests bring and have cached: "n", or "kxa-b" (k requests spread from a to b).
"""
import math

import numpy as np
import torch

own = False
DEV = "cuda"
_kernels = None


def listed():
    return [
        # one user: a small tree behind a short conversation, the attention of one layer; launches and latency count
        dict(name="tree_one", kind="tree", dtype="bfloat16", heads=16, kv_heads=8, dim=64, page=64, window=0, rows="12", contexts="1000"),
        # a served batch: trees of a few to two dozen tokens behind ragged contexts
        dict(name="tree_batch", kind="tree", dtype="bfloat16", heads=32, kv_heads=8, dim=64, page=64, window=0,
             rows="32x4-24", contexts="32x300-6000"),
        # larger trees behind long documents, heads of 128
        dict(name="tree_long", kind="tree", dtype="bfloat16", heads=32, kv_heads=8, dim=128, page=64, window=0,
             rows="8x24-64", contexts="8x4000-30000"),
        # the 32-bit mode, in which results are checked: windowed attention, small pages, one request new to the cache
        dict(name="tree_float32", kind="tree", dtype="float32", heads=16, kv_heads=4, dim=64, page=16, window=256,
             rows="4x1-21", contexts="4x0-900"),
        # a decode batch whose clients ask for twenty alternatives a token
        dict(name="score_decode", kind="logprobs", dtype="float32", rows=8, vocab=65536, top=20),
        # a prompt scored token by token, an odd vocabulary
        dict(name="score_prompt", kind="logprobs", dtype="float32", rows=2048, vocab=64401, top=5),
        # the tables of the served batch of trees
        dict(name="layout_trees", kind="layout", tree=True, page=64, rows="32x4-24", contexts="32x300-6000", spare=14),
        # the tables of a step full of prompt portions
        dict(name="layout_prompts", kind="layout", tree=False, page=64, rows="256x1-128", contexts="256x0-8000", spare=33),
        # which drafted tokens stand: a few requests, and a full batch of larger trees
        dict(name="accept_few", kind="accept", rows="4x6-12", vocab=65536),
        dict(name="accept_many", kind="accept", rows="256x8-64", vocab=65536),
        # the accepted rows into the pages of six layers: a few requests, and a full batch with heads of 128
        dict(name="commit_few", kind="commit", dtype="bfloat16", planes=6, kv_heads=8, dim=64, page=64, rows="4x6-12", contexts="4x100-500"),
        dict(name="commit_many", kind="commit", dtype="bfloat16", planes=6, kv_heads=8, dim=128, page=64, rows="64x8-32", contexts="64x20-400"),
    ]


def draw(rng):
    def log(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))

    def spread(k, lo, hi):
        a = log(max(lo, 1), hi)
        return "%dx%d-%d" % (k, a, log(a, hi))

    kind = rng.choice(["tree", "tree", "tree", "logprobs", "logprobs", "layout", "accept", "commit"])
    if kind == "tree":
        f32 = rng.random() < 0.25
        G = rng.choice([1, 2, 4, 8])
        c = dict(kind=kind, dtype="float32" if f32 else "bfloat16", heads=G * rng.choice([1, 2, 3, 4, 8] if G < 4 else [1, 2, 4]), kv_heads=G,
                 dim=rng.choice([64, 64, 128, 80, 32] if f32 else [64, 64, 64, 128, 128, 96]), page=rng.choice([16, 32, 64, 64]),
                 window=0 if rng.random() < 0.7 else log(16, 4096))
        S = log(1, 8 if f32 else 32)
        c["rows"] = spread(S, 1, 24 if f32 else 64)
        most = 1500 if f32 else min(30000, 60000 // S)
        c["contexts"] = "%dx0-%d" % (S, log(1, most)) if rng.random() < 0.3 else spread(S, 1, most)
        return c
    if kind == "logprobs":
        V = log(500, 131072)
        return dict(kind=kind, dtype="float32" if rng.random() < 0.75 else "bfloat16", rows=log(1, min(2048, 2048 * 64401 // V)), vocab=V,
                    top=rng.choice([0, 1, 5, 20, 32]))
    if kind == "layout":
        tree = rng.random() < 0.5
        S = log(1, 256)
        return dict(kind=kind, tree=tree, page=rng.choice([16, 32, 64]), rows=spread(S, 1, 64 if tree else 128), contexts="%dx0-%d" % (S, log(1, 8000)),
                    spare=rng.choice([0, rng.randint(1, 60)]))
    if kind == "accept":
        return dict(kind=kind, rows=spread(log(1, 256), 1, 64), vocab=log(8, 65536))
    return dict(kind=kind, dtype=rng.choice(["bfloat16", "bfloat16", "float32"]), planes=rng.randint(1, 6), kv_heads=rng.choice([1, 2, 4, 8]),
                dim=rng.choice([64, 64, 96, 128]), page=rng.choice([16, 32, 64]), rows=spread(log(1, 64), 1, 32), contexts="%s" % log(1, 400))


# ------------------------------------------------------------------------------------------------ sizes
def _counts(text, n=0):
    """The numbers that `text` stands for, spread ones in an order that mixes small and large; one number for all of `n`."""
    k, _, span = text.rpartition("x")
    a, _, b = span.partition("-")
    k, a, b = int(k) if k else max(n, 1), int(a), int(b or a)
    order = sorted(range(k), key=lambda i: (i * 0.6180339887) % 1.0)
    return [a + (b - a) * i // max(k - 1, 1) for i in order]


def _dtype(case):
    return torch.float32 if case["dtype"] == "float32" else torch.bfloat16


def _visible(case):
    """Pairs of (row, cached key) that attention has to look at, cached positions that it has to read."""
    q, ctx = _counts(case["rows"]), _counts(case["contexts"])
    seen = [min(c, case["window"] - 1) if case["window"] else c for c in ctx]
    return sum(n * (c + (n + 1) // 2) for n, c in zip(q, seen)), sum(seen)


def work(case):
    kind = case["kind"]
    if kind == "logprobs":
        es, R, V, k = 4 if case["dtype"] == "float32" else 2, case["rows"], case["vocab"], case["top"]
        return {"bytes": R * V * es + R * (16 + 8 * k), "flops": 5.0 * R * V}
    q = _counts(case["rows"])
    N, S = sum(q), len(q)
    if kind == "tree":
        es, G, D, H = 4 if case["dtype"] == "float32" else 2, case["kv_heads"], case["dim"], case["heads"]
        pairs, keys = _visible(case)
        return {"bytes": es * (keys * 2 * G * D + N * (2 * H * D + 2 * G * D)) + 4 * N * -(-max(q) // 32), "flops": 4.0 * pairs * H * D}
    if kind == "layout":
        ctx = _counts(case["contexts"])
        entries = S * -(-max(c + n for c, n in zip(ctx, q)) // case["page"])
        rows = N + case["spare"]
        return {"bytes": 4 * (2 * entries + 3 * rows + 7 * S + ((N + rows * -(-max(q) // 32)) if case["tree"] else 0)), "flops": 4.0 * rows}
    if kind == "accept":
        return {"bytes": 4 * (3 * N + 4 * S + 2 * S * max(q)), "flops": 2.0 * N}
    es = 4 if case["dtype"] == "float32" else 2
    kept = sum((n + 1) // 2 for n in q)                        # about half of a tree's longest path stands
    return {"bytes": 4 * es * case["planes"] * case["kv_heads"] * case["dim"] * kept, "flops": 0.0}


# ------------------------------------------------------------------------------------------------ inputs
def _ints(x):
    return torch.from_numpy(np.ascontiguousarray(x, dtype=np.int32)).to(DEV)


class _State:
    """What a step has in hand: the requests' lengths, on the host and on the device, and the tensors of its kind."""


def _trees(rng, q_lens):
    """Every row's parent among its request's rows (the first row has none): each hangs on one of the few rows before it, so that
    trees are some rows wide and many levels deep."""
    out = []
    for n in q_lens:
        i = np.arange(n)
        back = 1 + np.floor(rng.random(n) ** 2 * np.minimum(i, 6)).astype(np.int64)
        out.append(np.where(i == 0, -1, np.maximum(i - back, 0)))
    return out


def _levels(parents):
    """A tree's ancestors as a matrix (row sees column), and every row's depth."""
    n = len(parents)
    sees = np.zeros((n, n), dtype=bool)
    for i, p in enumerate(parents):
        if p >= 0:
            sees[i] = sees[p]
        sees[i, i] = True
    return sees, sees.sum(1) - 1


def _bits(sees, words):
    m = np.zeros((sees.shape[0], words * 32), dtype=np.uint64)
    m[:, :sees.shape[1]] = sees
    return (m.reshape(sees.shape[0], words, 32) << np.arange(32, dtype=np.uint64)).sum(2).astype(np.uint32).view(np.int32)


def prepare(case, seed):
    s = _State()
    s.case, s.kind = case, case["kind"]
    rng = np.random.default_rng(seed * 7919 + 11)
    g = torch.Generator(device=DEV).manual_seed(seed * 7919 + 17)
    if s.kind == "logprobs":
        R, V = case["rows"], case["vocab"]
        x = torch.randn((R, V), generator=g, device=DEV)
        x.mul_(2.5)
        for _ in range(8):                                         # a few tokens that stand out, as a trained model's rows have
            at = torch.randint(0, V, (R, 1), generator=g, device=DEV)
            x.scatter_(1, at, 8.0 + 6.0 * torch.rand((R, 1), generator=g, device=DEV))
        s.logits = x.to(_dtype(case))
        s.targets = torch.randint(0, V, (R,), generator=g, device=DEV, dtype=torch.int32)
        s.top = case["top"]
        return s
    s.q_lens = _counts(case["rows"])
    S, N = len(s.q_lens), sum(s.q_lens)
    s.S, s.N, s.T = S, N, max(s.q_lens)
    s.words = -(-s.T // 32)
    cu = np.concatenate([[0], np.cumsum(s.q_lens)])
    s.cu_q = _ints(cu)
    s.n_seqs, s.n_tokens, s.max_q_len = S, N, s.T
    trees = _trees(rng, s.q_lens)
    if s.kind != "layout" or case["tree"]:
        s.parents = _ints(np.concatenate(trees))
    if s.kind == "accept":
        V = case["vocab"]
        tokens, choices = rng.integers(0, V, N), rng.integers(0, V, N)
        for a, parents in zip(cu[:-1], trees):                     # most rows' choice is one of their drafted children
            for i in range(1, len(parents)):
                if rng.random() < 0.1:
                    tokens[a + i] = tokens[a + i - 1]                # (and some siblings draft the same token)
                if rng.random() < 0.6:
                    choices[a + parents[i]] = tokens[a + i]
        s.tokens, s.choices = _ints(tokens), _ints(choices)
        s.ctx_lens = _ints(rng.integers(0, 5000, S))
        return s
    s.ctx = _counts(case["contexts"], S)
    s.ctx_lens = _ints(s.ctx)
    s.page_size = ps = case["page"]
    s.max_kv_len = max(c + n for c, n in zip(s.ctx, s.q_lens))
    s.width = -(-s.max_kv_len // ps)
    held = [-(-(c + n) // ps) for c, n in zip(s.ctx, s.q_lens)]
    s.n_pages = sum(held) + 1
    ids = 1 + rng.permutation(sum(held))
    table = np.zeros((S, s.width), dtype=np.int64)
    at = 0
    for r, n in enumerate(held):
        table[r, :n] = ids[at:at + n]
        at += n
    if s.kind == "layout":
        s.slots = _ints(1 + rng.permutation(S + 7)[:S])
        rows = np.zeros((S + 8, s.width + 5), dtype=np.int64)       # the device's copy of every slot's block table
        rows[s.slots.cpu().numpy(), :s.width] = table
        s.page_rows, s.lens = _ints(rows), _ints(s.q_lens)
        s.rows = N + case["spare"]
        if case["tree"]:
            s.parents = torch.cat([s.parents, torch.full((case["spare"],), -1, dtype=torch.int32, device=DEV)])
        return s
    s.block_table = _ints(table)
    G, D, dt = case["kv_heads"], case["dim"], _dtype(case)
    first = np.repeat(cu[:-1], s.q_lens)
    s.seq_idx = _ints(np.repeat(np.arange(S), s.q_lens))
    if s.kind == "tree":
        H = case["heads"]
        levels = [_levels(p) for p in trees]
        s.tree_mask = _ints(np.concatenate([_bits(m, s.words) for m, _ in levels]))
        s.positions = _ints(np.concatenate([c + d for c, (_, d) in zip(s.ctx, levels)]))
        s.pages = torch.randn((s.n_pages, 2, G, ps, D), generator=g, device=DEV).to(dt)
        s.q = (2.0 * torch.randn((N, H * D), generator=g, device=DEV)).to(dt)
        qkv = torch.randn((N, (H + 2 * G) * D), generator=g, device=DEV).to(dt)
        s.k, s.v = qkv[:, H * D:(H + G) * D], qkv[:, (H + G) * D:]     # (rows of the projection)
        s.scale, s.window = D ** -0.5, case["window"] or None
        return s
    pos = np.repeat(s.ctx, s.q_lens) + np.arange(N) - first
    s.kv_slots = _ints(table[np.repeat(np.arange(S), s.q_lens), pos // ps] * ps + pos % ps)
    L = case["planes"]
    s.pages = torch.randn((L, s.n_pages, 2, G, ps, D), generator=g, device=DEV).to(dt)
    s.k = torch.randn((L, N, G * D), generator=g, device=DEV).to(dt)
    s.v = torch.randn((L, N, G * D), generator=g, device=DEV).to(dt)
    counts = [(n + 1) // 2 for n in s.q_lens]
    path = np.full((S, max(counts)), -1, dtype=np.int64)
    for r, (n, c) in enumerate(zip(s.q_lens, counts)):
        path[r, :c] = cu[r] + np.sort(np.concatenate([[0], 1 + rng.permutation(n - 1)[:c - 1]]).astype(np.int64))
    s.path, s.counts = _ints(path), _ints(counts)
    return s


# ------------------------------------------------------------------------------------------------ the operators
def run(s):
    global _kernels
    if own:
        if _kernels is None:
            import zig_ai_b200  # noqa: F401
            from zig_ai_b200.kernels import ops
            _kernels = ops
        ops = _kernels
        if s.kind == "tree":
            c = s.case
            return ops.tree_attention(s.q, s.k, s.v, s, s, c["heads"], c["kv_heads"], c["dim"], s.scale, s.window)
        if s.kind == "logprobs":
            return ops.token_logprobs(s.logits, s.targets, s.top)._asdict()
        if s.kind == "layout":
            parents = s.parents if s.case["tree"] else None
            return {k: v for k, v in ops.step_layout(s.lens, s.ctx_lens, s.slots, s.page_rows, s.page_size, s.rows, s.width, parents,
                                                     s.T if s.case["tree"] else 0)._asdict().items() if v is not None}
        if s.kind == "accept":
            return ops.accept_drafts(s.choices, s.tokens, s.parents, s, s.T)._asdict()
        ops.commit_drafts(s.k, s.v, s.path, s.counts, s, s.pages)
        return s.pages
    return {"tree": _tree, "logprobs": _logprobs, "layout": _layout, "accept": _accept, "commit": _commit}[s.kind](s)


def _padded_rows(s):
    """[S, T]: the row of each request's i-th token, and whether there is one."""
    i = torch.arange(s.T, device=DEV)
    rows = s.cu_q[:-1, None].long() + i
    return rows.clamp(max=s.N - 1), rows < s.cu_q[1:, None]


def _tree(s):
    c = s.case
    H, G, D, S, T = c["heads"], c["kv_heads"], c["dim"], s.S, s.T
    rows, real = _padded_rows(s)
    q = s.q[rows].view(S, T, G, H // G, D).permute(0, 2, 1, 3, 4).reshape(S, G, T * (H // G), D).float()
    kv = s.pages[s.block_table.long()]                              # [S, width, 2, G, page, D]
    k, v = (kv[:, :, i].permute(0, 2, 1, 3, 4).reshape(S, G, -1, D).float() for i in (0, 1))
    k = torch.cat([k, s.k[rows].view(S, T, G, D).transpose(1, 2).float()], 2)
    v = torch.cat([v, s.v[rows].view(S, T, G, D).transpose(1, 2).float()], 2)
    L = s.width * s.page_size
    pos = s.positions[rows]                                         # [S, T]
    at = torch.arange(L, device=DEV)
    cached = (at < s.ctx_lens[:, None]).unsqueeze(1).expand(S, T, L)
    j = torch.arange(T, device=DEV)
    drafted = (s.tree_mask[rows][:, :, j // 32] >> (j % 32) & 1).bool() & real[:, None, :]
    if s.window:
        cached = cached & (at > pos[:, :, None] - s.window)
        drafted = drafted & (pos[:, None, :] > pos[:, :, None] - s.window)
    sees = torch.cat([cached, drafted], 2)[:, None, :, None, :].expand(S, G, T, H // G, L + T).reshape(S, G, T * (H // G), L + T)
    a = torch.where(sees, (q @ k.transpose(2, 3)) * s.scale, float("-inf"))
    top = a.amax(-1, keepdim=True)
    a = torch.exp(a - torch.where(top == float("-inf"), 0.0, top))
    total = a.sum(-1, keepdim=True)
    o = (a @ v) / torch.where(total == 0, 1.0, total)
    return o.view(S, G, T, H // G, D).permute(0, 2, 1, 3, 4).reshape(S, T, H * D)[real].to(s.q.dtype)


def _logprobs(s):
    x = s.logits.float() + 0.0
    V = x.shape[1]
    top = x.amax(1, keepdim=True)
    d = x - top
    e = torch.exp(d)
    z = e.sum(1)
    log_z = torch.log(z)
    t = s.targets.long()[:, None]
    xt = x.gather(1, t)
    at = torch.arange(V, device=DEV)
    out = {"logprobs": d.gather(1, t)[:, 0] - log_z,
           "entropy": log_z - (e * d).sum(1) / z,
           "ranks": ((x > xt).sum(1) + ((x == xt) & (at < t)).sum(1)).int()}
    bits = x.view(torch.int32)
    key = ((bits ^ (bits >> 31 & 0x7fffffff)).long() << 32) + (V - 1 - at)     # by value, then by the lower index
    best = key.topk(s.top, 1).values
    out["top_ids"] = (V - 1 - (best & 0xffffffff)).int()
    out["top_logprobs"] = d.gather(1, out["top_ids"].long()) - log_z[:, None]
    return out


def _ancestors(parents, T):
    """[S, T, T] of zeros and ones: row i of a tree sees row j (itself and what it hangs on), by squaring "is i or i's parent"."""
    j = torch.arange(T, device=parents.device)
    near = (parents[:, :, None] == j) | (j[:, None] == j)
    near = near.float()
    for _ in range(max(T - 1, 1).bit_length()):
        near = (near @ near).clamp(max=1.0)
    return near


def _layout(s):
    ps, S = s.page_size, s.S
    zero = torch.zeros(1, dtype=torch.int32, device=DEV)
    cu = torch.cat([zero, s.lens.cumsum(0, dtype=torch.int32), torch.full_like(zero, s.rows)])
    row = torch.arange(s.rows, device=DEV, dtype=torch.int32)
    seq = torch.searchsorted(cu[1:-1], row, right=True)
    i = row - cu[seq]
    ctx = torch.cat([s.ctx_lens, zero])
    tables = torch.cat([s.page_rows[s.slots.long(), :s.width], torch.zeros((1, s.width), dtype=torch.int32, device=DEV)])
    pos = torch.where(seq < S, ctx[seq] + i, i % (s.width * ps))
    slots = torch.where(seq < S, tables[seq, (pos // ps).long()] * ps + pos % ps, -1)
    out = {"cu_q": cu, "ctx_lens": ctx, "positions": pos, "seq_idx": seq.int(), "kv_slots": slots, "block_tables": tables}
    if s.case["tree"]:
        rows, real = _padded_rows(s)
        parents = torch.where(real, s.parents[rows], -1)
        sees = _ancestors(parents, s.T)
        depth = sees.sum(2).int() - 1
        j = torch.arange(s.words * 32, device=DEV)
        wide = torch.zeros((S, s.T, s.words * 32), dtype=torch.int64, device=DEV)
        wide[:, :, :s.T] = sees.long()
        bits = (wide << (j % 32)).view(S, s.T, s.words, 32).sum(3)
        bits = torch.where(bits >= 2 ** 31, bits - 2 ** 32, bits).int()
        mask = torch.zeros((s.rows, s.words), dtype=torch.int32, device=DEV)
        mask[:s.N] = bits[real]
        pos[:s.N] = (s.ctx_lens[:, None] + depth)[real]
        out["tree_mask"] = mask
    return out


def _accept(s):
    S, T = s.S, s.T
    rows, real = _padded_rows(s)
    parents = torch.where(real, s.parents[rows], -1)
    tokens, choices = s.tokens[rows], s.choices[rows]
    wanted = choices.gather(1, parents.clamp(min=0).long())
    j = torch.arange(T, device=DEV)
    hit = real & ((parents >= 0) & (tokens == wanted) | (j == 0))
    twin = (parents[:, :, None] == parents[:, None, :]) & (tokens[:, :, None] == tokens[:, None, :]) & (j[None, :] < j[:, None]) & hit[:, None, :]
    hit = hit & ~twin.any(2)                                         # the first of several children with one token
    stands = real & ((_ancestors(parents, T) @ (~hit).float()[:, :, None])[:, :, 0] == 0)
    counts = stands.sum(1)
    order = torch.where(stands, j, T).sort(1).values
    kept = order < T
    order = order.clamp(max=T - 1)
    path = torch.where(kept, rows.gather(1, order), -1).int()
    chosen = torch.where(kept, choices.gather(1, order), -1)
    return {"counts": counts.int(), "path": path, "tokens": chosen, "ctx_lens": s.ctx_lens + counts.int()}


def _commit(s):
    L, _, _, G, ps, D = s.pages.shape
    P = s.path.shape[1]
    i = torch.arange(P, device=DEV)
    kept = i < s.counts[:, None]
    slot = s.kv_slots[(s.cu_q[:-1, None].long() + i).clamp(max=s.N - 1)][kept].long()
    src = s.path[kept].long()
    s.pages[:, slot // ps, 0, :, slot % ps] = s.k[:, src].view(L, -1, G, D).transpose(0, 1)
    s.pages[:, slot // ps, 1, :, slot % ps] = s.v[:, src].view(L, -1, G, D).transpose(0, 1)
    return s.pages


# ------------------------------------------------------------------------------------------------ the same in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if s.kind == "logprobs":
        lp, ent, top = [], [], []
        for x, t in zip(s.logits.split(128), s.targets.split(128)):
            p = torch.log_softmax(x.double(), 1)
            lp.append(p.gather(1, t.long()[:, None])[:, 0])
            ent.append(-(p.exp() * p).sum(1))
            top.append(p.topk(s.top, 1).values)
        return {"logprobs": torch.cat(lp), "entropy": torch.cat(ent), "ranks": None, "top_ids": None, "top_logprobs": torch.cat(top)}
    if s.kind == "commit":
        pages, cu, slots = s.pages.double(), s.cu_q.tolist(), s.kv_slots.tolist()
        G, D = case["kv_heads"], case["dim"]
        for r, n in enumerate(s.counts.tolist()):
            for i, row in enumerate(s.path[r, :n].tolist()):
                page, at = divmod(slots[cu[r] + i], s.page_size)
                for which, rows in ((0, s.k), (1, s.v)):
                    pages[:, page, which, :, at] = rows[:, row].double().view(-1, G, D)
        return pages
    if s.kind != "tree":
        return None
    H, G, D, ps = case["heads"], case["kv_heads"], case["dim"], s.page_size
    cu, out = s.cu_q.tolist(), []
    for r, (n, c) in enumerate(zip(s.q_lens, s.ctx)):
        a, b = cu[r], cu[r + 1]
        kv = s.pages[s.block_table[r, :max(-(-c // ps), 1)].long()].double().permute(1, 2, 0, 3, 4).reshape(2, G, -1, D)[:, :, :c]
        pos = torch.cat([torch.arange(c, device=DEV), s.positions[a:b].long()])
        drafted = torch.stack([s.k[a:b], s.v[a:b]]).double().view(2, n, G, D).transpose(1, 2)
        kv = torch.cat([kv, drafted], 2)
        for i in range(n):
            words = s.tree_mask[a + i].tolist()
            sees = torch.tensor([True] * c + [bool(words[j // 32] >> (j % 32) & 1) for j in range(n)], device=DEV)
            if case["window"]:
                sees &= pos > int(pos[c + i]) - case["window"]
            q = s.q[a + i].double().view(G, H // G, D)
            p = torch.softmax((q @ kv[0].transpose(1, 2) * s.scale).masked_fill(~sees, float("-inf")), -1)
            out.append((p @ kv[1]).reshape(H * D))
    return torch.stack(out)
