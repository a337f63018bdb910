"""The kernels of a step that checks drafted tokens (step tables, tree attention, log probabilities, the accepted path, the accepted
rows' keys and values) against plain versions in 64 bits (tests/ref_ops.py)."""
import random
from types import SimpleNamespace

import pytest
import torch

import ref_ops

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def ops():
    from zig_ai_b200.kernels import ops as o
    return o


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def make_parents(g, n, shape="mixed"):
    if shape == "chain":
        return [i - 1 for i in range(n)]
    if n == 0:
        return []
    if shape == "star":
        return [-1] + [0] * (n - 1)
    if shape == "forest":
        return [-1 if i == 0 or g.random() < 0.3 else g.randrange(i) for i in range(n)]
    return [-1] + [max(i - 1 - g.randrange(4), 0) for i in range(1, n)]


def make_masks(parents_by_span, words):
    rows, depths = [], []
    for parents in parents_by_span:
        bits, depth = [], []
        for i, p in enumerate(parents):
            bits.append((bits[p] if p >= 0 else 0) | 1 << i)
            depth.append(depth[p] + 1 if p >= 0 else 0)
        rows += [[b >> 32 * w & 0xffffffff for w in range(words)] for b in bits]
        depths.append(depth)
    return torch.tensor(rows, dtype=torch.int64).to(torch.int32).view(-1, words).cuda(), depths


def make_tree_step(q_lens, ctx, H, G, D, ps, dtype, seed, shape="mixed", extra_words=0, poison=float("nan"), packed=True):
    """A step of trees behind random block tables; everything of the pages that no row may look at is `poison`."""
    g, t = random.Random(seed), torch.Generator(device="cuda").manual_seed(seed)
    S, N = len(q_lens), sum(q_lens)
    parents = [make_parents(g, n, shape) for n in q_lens]
    words = max(-(-max(q_lens + [1]) // 32), 1) + extra_words
    mask, depths = make_masks(parents, words)
    width = max(max(-(-(c + n) // ps) for c, n in zip(ctx, q_lens)), 1)
    held = [-(-c // ps) for c in ctx]
    ids = list(range(1, sum(held) + 3))
    g.shuffle(ids)
    table, pages = [], torch.full((sum(held) + 3, 2, G, ps, D), poison, dtype=dtype, device="cuda")
    for c, n in zip(ctx, held):
        row = [ids.pop() for _ in range(n)]
        for j, p in enumerate(row):
            m = min(ps, c - j * ps)
            pages[p, :, :, :m] = torch.randn((2, G, m, D), generator=t, device="cuda").to(dtype)
        table.append(row + [0] * (width - n))
    q = (2 * torch.randn((N, H * D), generator=t, device="cuda")).to(dtype)
    qkv = torch.randn((N, (H + 2 * G) * D), generator=t, device="cuda").to(dtype)
    k, v = qkv[:, H * D:(H + G) * D], qkv[:, (H + G) * D:]
    if packed:
        k, v = k.contiguous(), v.contiguous()
    cu = [0]
    for n in q_lens:
        cu.append(cu[-1] + n)
    step = SimpleNamespace(cu_q=ints(cu), ctx_lens=ints(ctx), positions=ints([c + d for c, ds in zip(ctx, depths) for d in ds]), tree_mask=mask,
                           n_seqs=S, n_tokens=N, max_q_len=max(q_lens), q_lens=q_lens)
    return q, k, v, step, SimpleNamespace(pages=pages, block_table=ints(table), page_size=ps), parents


def close(got, q, k, v, step, cache, H, G, D, scale, window):
    """Against 64 bits.  With u the half step of 32 bits (2^-24) a score is off by at most d = (D + 4) u sum|q k| scale (products and sums in any
    order) and a few u of itself in the exponential's argument; a weight by a factor e^(2 d) and 8 u, the sums by the number of
    keys times u: |o - o64| <= sum p|v| (2 d + (keys + 16) u), and in bfloat16 half a step of 2^-8 for the weights (times sum
    p|v|) and one for the result."""
    want = ref_ops.tree_attention(q, k, v, step, cache, H, G, D, scale, window)
    exact = ref_ops.tree_attention(q.double(), k, v, step, cache, H, G, D, scale, window)
    size = ref_ops.tree_attention(q.double(), k, v, step, cache, H, G, D, scale, window, absolute=True)
    assert got.dtype == q.dtype and got.shape == want.shape
    u, keys = 2.0 ** -24, max(int(step.ctx_lens.max()), 0) + step.max_q_len
    kmax = max(float(cache.pages[:, 0].double().nan_to_num().abs().max()), float(k.double().nan_to_num().abs().max()))
    score = float(q.double().abs().view(-1, D).sum(1).max()) * kmax * scale
    bound = size * (2 * (D + 8) * u * score + (keys + 16) * u)
    if q.dtype == BF16:
        bound = bound + 2.0 ** -8 * size + 2.0 ** -8 * exact.abs()
    over = (got.double() - exact).abs() - bound
    assert torch.isfinite(got).all()
    assert float(over.max()) <= 0, (float(over.max()), float((got.double() - exact).abs().max()))


TREES = [
    # q_lens, ctx, H, G, D, page, window
    ([1], [0], 2, 2, 64, 16, None),                            # one row that sees itself alone
    ([1], [1], 4, 1, 64, 16, None),
    ([5], [63], 8, 2, 64, 64, None),
    ([12], [1000], 16, 8, 64, 64, None),
    ([3, 1, 9, 24, 2], [64, 0, 129, 500, 17], 8, 2, 64, 16, None),
    ([33, 64, 65], [100, 31, 640], 8, 2, 64, 32, None),        # masks of several words, tiles of pairs that end inside a row's heads
    ([40], [300], 3, 1, 64, 8, None),                          # three heads share a key/value head
    ([70, 3], [257, 2000], 16, 2, 128, 64, None),
    ([7, 11], [333, 90], 4, 4, 128, 16, 50),                   # windows: inside the cache, inside the tree
    ([20, 33], [400, 3], 8, 4, 64, 16, 7),
    ([6, 2], [64, 65], 4, 2, 96, 16, None),
    ([9, 4], [130, 5], 6, 2, 32, 4, 40),
    ([5, 8], [77, 12], 6, 3, 80, 16, None),                    # the general kernel's head sizes
    ([4, 3], [40, 19], 2, 1, 13, 5, None),
    ([3], [21], 2, 2, 320, 8, 9),
    ([130], [40], 2, 1, 64, 16, None),                         # a large tree
]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("q_lens,ctx,H,G,D,ps,window", TREES)
def test_tree_attention(dtype, q_lens, ctx, H, G, D, ps, window):
    for shape in ("mixed", "forest"):
        q, k, v, step, cache, _ = make_tree_step(list(q_lens), list(ctx), H, G, D, ps, dtype, 7, shape, packed=shape == "mixed")
        got = ops().tree_attention(q, k, v, step, cache, H, G, D, D ** -0.5, window)
        close(got, q, k, v, step, cache, H, G, D, D ** -0.5, window)
    assert ops().read_status() == 0


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("q_lens,ctx,group", [([1], [0], 1), ([1], [128], 2), ([5], [127], 4), ([64, 3], [1000, 129], 4), ([33, 0, 16, 7], [5000, 3, 0, 640], 4),
                                              ([128, 40], [300, 2500], 4), ([1] * 40, [7 * i for i in range(40)], 1), ([24, 9] * 17, [900, 0] * 17, 8),
                                              ([60], [20000], 4), ([2, 2], [70000, 1], 2)])
@pytest.mark.parametrize("shape", ["mixed", "forest"])
def test_tree_attention_in_shares(D, q_lens, ctx, group, shape):
    """The tcgen05 kernel: shares that begin and end inside a unit, units of one and two turns, requests without rows or without a cache."""
    H, G = 2 * group, 2
    q, k, v, step, cache, _ = make_tree_step(list(q_lens), list(ctx), H, G, D, 64, BF16, 13, shape, extra_words=1, packed=shape == "mixed")
    got = ops().tree_attention(q, k, v, step, cache, H, G, D, D ** -0.5, impl="tcgen05")
    close(got, q, k, v, step, cache, H, G, D, D ** -0.5, None)
    assert ops().read_status() == 0


@pytest.mark.parametrize("dtype,impl", [(F32, None), (BF16, "general"), (BF16, "mma")])
@pytest.mark.parametrize("splits", [1, 2, 4, 8, 16])
@pytest.mark.parametrize("D,group,n", [(64, 2, 5), (64, 4, 8), (64, 4, 14), (128, 4, 30), (128, 8, 2)])
def test_tree_attention_by_every_split(dtype, impl, splits, D, group, n):
    """Every number of blocks that share a tile's keys, more than there are tiles among them."""
    q, k, v, step, cache, _ = make_tree_step([n, 1, n], [700, 3, 129], 2 * group, 2, D, 16, dtype, 11, extra_words=2)
    got = ops().tree_attention(q, k, v, step, cache, 2 * group, 2, D, D ** -0.5, impl=impl, splits=splits)
    close(got, q, k, v, step, cache, 2 * group, 2, D, D ** -0.5, None)


IMPLS = [(F32, None, 1), (F32, None, 4), (BF16, "general", 1), (BF16, "general", 4), (BF16, "mma", 1), (BF16, "mma", 4), (BF16, "tcgen05", None)]


@pytest.mark.parametrize("dtype,impl,splits", IMPLS)
def test_rows_that_see_nothing_and_empty_spans(dtype, impl, splits):
    """A mask without bits over an empty cache gives zeros; spans without rows take no part."""
    q, k, v, step, cache, _ = make_tree_step([4, 6, 3], [0, 50, 0], 4, 2, 64, 16, dtype, 3)
    step.tree_mask[1] = 0
    step.tree_mask[10:13] = 0
    step.cu_q = ints([0, 4, 4, 10, 13, 13])                    # (a span without rows has a length and a table all the same)
    step.ctx_lens, step.n_seqs = ints([0, 900, 50, 0, 7]), 5
    cache.block_table = cache.block_table[[0, 1, 1, 2, 1]].contiguous()
    got = ops().tree_attention(q, k, v, step, cache, 4, 2, 64, 0.125, impl=impl, splits=splits)
    close(got, q, k, v, step, cache, 4, 2, 64, 0.125, None)
    assert not got[[1, 10, 11, 12]].any()


@pytest.mark.parametrize("dtype,impl", [(F32, None), (BF16, "general"), (BF16, "mma"), (BF16, "tcgen05")])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_what_is_not_finite_reaches_the_rows_that_see_it_alone(dtype, impl, bad):
    H, G, D = 4, 2, 64
    q, k, v, step, cache, parents = make_tree_step([9, 70], [100, 40], H, G, D, 16, dtype, 5)
    want = ops().tree_attention(q, k, v, step, cache, H, G, D, 0.125, impl=impl, splits=2)
    k, v = k.clone(), v.clone()
    k[4] = bad                                              # row 4 of the first tree, row 60 of the second
    v[9 + 60, :D] = bad
    got = ops().tree_attention(q, k, v, step, cache, H, G, D, 0.125, impl=impl, splits=2)
    sees = ref_ops._bits(step.tree_mask, 70)
    hit = torch.zeros((79, H, D), dtype=torch.bool, device="cuda")
    hit[:9][sees[:9, 4]] = True
    hit[9:, :H // G][sees[9:, 60]] = True                     # (the first key/value head's query heads)
    hit = hit.view(79, -1)
    assert torch.equal(got[~hit], want[~hit])
    assert not torch.isfinite(got[hit]).any()
    if impl == "tcgen05":                                    # (takes no window)
        return
    # a window's edge inside a tile of cached keys
    q, k, v, step, cache, _ = make_tree_step([6], [90], H, G, D, 16, dtype, 6, "chain")
    clean = ops().tree_attention(q, k, v, step, cache, H, G, D, 0.125, 20, impl=impl, splits=1)
    page, off = int(cache.block_table[0, 72 // 16]), 72 % 16
    cache.pages[page, 1, :, off] = bad                       # position 72: rows at 90 and 91 see it (72 > 91 - 20), those behind do not
    got = ops().tree_attention(q, k, v, step, cache, H, G, D, 0.125, 20, impl=impl, splits=1)
    assert torch.equal(got[2:], clean[2:]) and not torch.isfinite(got[:2]).any()


@pytest.mark.parametrize("dtype,impl", [(F32, None), (BF16, "general"), (BF16, "mma"), (BF16, "tcgen05")])
@pytest.mark.parametrize("grow", [0.02, 6.0, 40.0])
def test_scores_that_grow_along_the_keys(dtype, impl, grow):
    """The running maximum moves tile by tile, by little or by hundreds; the last keys, or the drafted rows, outweigh all before them."""
    H, G, D = 8, 2, 64
    for ctx in (700, 300):
        q, k, v, step, cache, _ = make_tree_step([9, 40], [ctx, 1100], H, G, D, 16, dtype, 5)
        q[:, ::64] = 8.0                                    # (every head's first column)
        for s in range(2):
            n = int(step.ctx_lens[s])
            table = cache.block_table[s].tolist()
            for j in range(0, n, 5):
                cache.pages[table[j // 16], 0, :, j % 16, 0] = grow * j / 128
        k[4, ::64] = grow * 9
        got = ops().tree_attention(q, k, v, step, cache, H, G, D, 0.125, impl=impl)
        # (scores of hundreds: their rounding is what the bound of `close` is made of, with the largest of all of them)
        close(got, q, k, v, step, cache, H, G, D, 0.125, None)
    assert ops().read_status() == 0


def test_spans_longer_than_the_step_says_raise_the_status_word():
    for n, said, impl, dtype in ((9, 2, "mma", BF16), (40, 16, "mma", BF16), (130, 100, "tcgen05", BF16), (30, 3, None, F32)):
        q, k, v, step, cache, _ = make_tree_step([n, n], [40, 100], 4, 2, 64, 16, dtype, 5)
        step.max_q_len = n if said == 100 else said
        if impl == "tcgen05":
            step.max_q_len = said
        ops().tree_attention(q, k, v, step, cache, 4, 2, 64, 0.125, impl=impl)
        assert ops().read_status() == 64, (n, said, impl)


def test_tree_attention_large_offsets():
    """A pool whose later pages lie beyond 2^31 elements."""
    H, G, D, ps = 4, 2, 64, 64
    per_page = 2 * G * ps * D
    n_pages = (1 << 31) // per_page + 40
    pages = torch.empty((n_pages, 2, G, ps, D), dtype=BF16, device="cuda")
    q, k, v, step, cache, _ = make_tree_step([5, 3], [200, 130], H, G, D, ps, BF16, 9)
    used = cache.pages.shape[0]
    pages[-used:] = cache.pages
    pages[0] = float("nan")
    want = ops().tree_attention(q, k, v, step, cache, H, G, D, 0.125)
    far = SimpleNamespace(pages=pages, page_size=ps, block_table=torch.where(cache.block_table > 0, cache.block_table + n_pages - used, 0).int())
    for impl in ("mma", "general", "tcgen05"):
        near = ops().tree_attention(q, k, v, step, cache, H, G, D, 0.125, impl=impl)
        assert torch.equal(ops().tree_attention(q, k, v, step, far, H, G, D, 0.125, impl=impl), near)
    assert want.isfinite().all()


def test_bad_pages_raise_the_status_word():
    q, k, v, step, cache, _ = make_tree_step([5, 3], [200, 130], 4, 2, 64, 16, BF16, 9, poison=0.0)
    good = ops().tree_attention(q, k, v, step, cache, 4, 2, 64, 0.125)
    assert ops().read_status() == 0
    bt = cache.block_table.clone()
    bt[0, 3] = cache.pages.shape[0]
    for impl in ("mma", "general", "tcgen05"):
        got = ops().tree_attention(q, k, v, step, SimpleNamespace(pages=cache.pages, block_table=bt, page_size=16), 4, 2, 64, 0.125, impl=impl)
        assert ops().read_status() == 4
        assert torch.isfinite(got).all() and (impl != "mma" or torch.equal(got[5:], good[5:]))
    narrow = SimpleNamespace(pages=cache.pages, block_table=cache.block_table[:, :5].contiguous(), page_size=16)
    for impl in ("mma", "general", "tcgen05"):
        ops().tree_attention(q, k, v, step, narrow, 4, 2, 64, 0.125, impl=impl)
        assert ops().read_status() == 16
    step.cu_q = ints([0, 5, 99])
    step.n_seqs = 2
    for impl in ("mma", "general", "tcgen05"):
        ops().tree_attention(q, k, v, step, cache, 4, 2, 64, 0.125, impl=impl)
        assert ops().read_status() == 32


def test_unaligned_rows_take_the_general_kernel():
    q, k, v, step, cache, _ = make_tree_step([5, 3], [20, 130], 4, 2, 64, 16, BF16, 9)
    wide = torch.zeros((8, 2 * 64 + 3), dtype=BF16, device="cuda")
    wide[:, 1:129] = k
    got = ops().tree_attention(q, wide[:, 1:129], v, step, cache, 4, 2, 64, 0.125)
    close(got, q, k, v, step, cache, 4, 2, 64, 0.125, None)
    with pytest.raises(ops().KernelError, match="16-byte"):
        ops().tree_attention(q, wide[:, 1:129], v, step, cache, 4, 2, 64, 0.125, impl="mma")


def test_tree_attention_refuses():
    q, k, v, step, cache, _ = make_tree_step([5, 3], [20, 130], 4, 2, 64, 16, BF16, 9)
    o = ops()

    def call(**kw):
        a = dict(q=q, k=k, v=v, step=step, cache=cache, heads=4, kv_heads=2, head_dim=64, scale=0.125, window=None)
        a.update(kw)
        with pytest.raises(o.KernelError):
            o.tree_attention(**a)

    def but(ns, **kw):
        return SimpleNamespace(**{**vars(ns), **kw})

    call(kv_heads=3)
    call(q=q.float())
    call(k=k[:, :64])
    call(v=v[:4])
    call(scale=0.0)
    call(scale=float("nan"))
    call(window=0)
    call(step=but(step, tree_mask=None))
    call(step=but(step, tree_mask=step.tree_mask[:3]))
    call(step=but(step, tree_mask=step.tree_mask.long()))
    call(step=but(step, ctx_lens=step.ctx_lens[:1]))
    call(step=but(step, n_tokens=9))
    call(step=but(step, positions=step.positions[:5]))
    call(cache=but(cache, pages=cache.pages.float()))
    call(cache=but(cache, page_size=8))
    call(cache=but(cache, block_table=cache.block_table[:1]))
    call(q=q.cpu())
    call(splits=3 * 16)
    empty = but(step, n_tokens=0, tree_mask=step.tree_mask[:0], positions=step.positions[:0], cu_q=ints([0, 0, 0]))
    assert o.tree_attention(q[:0], k[:0], v[:0], empty, cache, 4, 2, 64, 0.125).shape == (0, 256)


# ------------------------------------------------------------------------------------------------ log probabilities
def check_logprobs(x, t, top, **kw):
    got, want = ops().token_logprobs(x, t, top, **kw), ref_ops.token_logprobs(x, t, top)
    assert torch.equal(got.ranks, want.ranks) and torch.equal(got.top_ids, want.top_ids)
    # 32 bits: differences from the maximum are off by half a step of themselves, at most 2^-24 of the row's spread; ln z by the relative error of
    # z (a few steps of the exponential, V / 512 terms a thread one after the other); the entropy by that of u as well
    spread = (x.double().amax(1) - torch.where(x.double() == float("-inf"), x.double().amax(1, keepdim=True), x.double()).amin(1)).clamp(1.0, 200.0)
    tol = 2.0 ** -24 * (spread * 4 + 8 + x.shape[1] / 128)
    for a, b in ((got.logprobs, want.logprobs), (got.entropy, want.entropy)):
        far = (a.double() - b).abs()
        assert bool(((far <= tol + 2.0 ** -23 * b.abs()) | (a.double() == b)).all()), float(far.max())
    far = (got.top_logprobs.double() - want.top_logprobs).abs()
    assert bool(((far <= tol[:, None] + 2.0 ** -23 * want.top_logprobs.abs()) | (got.top_logprobs.double() == want.top_logprobs)).all())
    return got


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("R,V,top", [(1, 1, 0), (1, 1, 1), (3, 2, 2), (2, 31, 5), (5, 32, 32), (1, 777, 20), (4, 8191, 1), (3, 8192, 32), (2, 8193, 5),
                                     (7, 65536, 20), (33, 50001, 3), (160, 20003, 8), (400, 3001, 0), (1, 200001, 32)])
def test_token_logprobs(dtype, R, V, top):
    g = torch.Generator(device="cuda").manual_seed(R * 1000 + V)
    x = (3 * torch.randn((R, V), generator=g, device="cuda")).to(dtype)
    t = torch.randint(0, V, (R,), generator=g, device="cuda", dtype=torch.int32)
    t[0] = V - 1
    check_logprobs(x, t, top)


@pytest.mark.parametrize("blocks", [1, 2, 4, 8, 16])
@pytest.mark.parametrize("V", [5, 70000, 33333])
def test_token_logprobs_by_every_split(blocks, V):
    g = torch.Generator(device="cuda").manual_seed(V)
    x = 2 * torch.randn((3, V), generator=g, device="cuda")
    check_logprobs(x, ints([0, V - 1, V // 2]), 5, blocks=blocks)
    assert torch.equal(ops().token_logprobs(x, ints([0, V - 1, V // 2]), 5, blocks=blocks).logprobs,
                       ops().token_logprobs(x, ints([0, V - 1, V // 2]), 5, blocks=blocks).logprobs)


@pytest.mark.parametrize("blocks", [0, 1, 4])
def test_token_logprobs_of_unusual_rows(blocks):
    """Ties, rows that ascend or descend, masked tokens (-inf and the type's lowest value), a single token left."""
    V = 40000
    j = torch.arange(V, device="cuda").float()
    low = torch.finfo(F32).min
    rows = [torch.zeros(V, device="cuda"), j / V, -j / V, (j % 7).clone(), torch.full((V,), low, device="cuda")]
    masked = torch.full((V,), float("-inf"), device="cuda")
    masked[[39, 20000, V - 1]] = torch.tensor([1.0, 1.0, -2.0], device="cuda")
    lowest = torch.full((V,), low, device="cuda")
    lowest[[5, 30000]] = torch.tensor([2.0, 3.0], device="cuda")
    only = torch.full((V,), float("-inf"), device="cuda")
    only[17] = -4.0
    signed = torch.where(j % 2 == 0, -0.0, 0.0)
    peak = torch.randn(V, device="cuda")
    peak[12345] = 120.0
    x = torch.stack(rows + [masked, lowest, only, signed, peak])
    for t in ([0, V - 1, V - 1, 6, 100, 20000, 5, 17, 1, 12345], [V - 1, 0, 0, 13, 0, 39, 30000, 17, 0, 1]):
        check_logprobs(x, ints(t), 20, blocks=blocks)
    got = ops().token_logprobs(x, ints([-1] * 10), 3, blocks=blocks)
    assert got.logprobs.tolist() == [0.0] * 10 and got.ranks.tolist() == [-1] * 10
    masked_token = ops().token_logprobs(x[5:6], ints([3]), 0, blocks=blocks)
    assert masked_token.logprobs.tolist() == [float("-inf")] and masked_token.ranks.tolist() == [3 + 3]       # three tokens that can come, three before it that cannot
    assert ops().read_status() == 0


def test_token_logprobs_of_rows_without_a_distribution():
    V = 9000
    x = torch.randn((4, V), device="cuda")
    x[0] = float("-inf")
    x[1, 4000] = float("inf")
    x[2, 17] = float("nan")
    got = ops().token_logprobs(x, ints([1, 2, 3, 4]), 4)
    assert torch.isnan(got.logprobs[[0, 1, 2]]).all() and torch.isnan(got.entropy[[0, 1, 2]]).all()
    assert bool(((got.top_ids >= 0) & (got.top_ids < V)).all())
    assert torch.isfinite(got.logprobs[3])


def test_token_logprobs_of_strided_rows_and_tokens_outside():
    g = torch.Generator(device="cuda").manual_seed(1)
    for dtype in (F32, BF16):
        wide = torch.randn((6, 5003), generator=g, device="cuda").to(dtype)
        check_logprobs(wide[:, 2:4500], ints([0, 1, 2, 3, 4, 4497]), 6)
        check_logprobs(wide[::2, 1:], ints([5, 6, 7]), 6)
    x = torch.randn((3, 100), generator=g, device="cuda")
    got = ops().token_logprobs(x, ints([100, 4, -2]), 2)
    assert ops().read_status() == 2
    assert got.ranks.tolist()[::2] == [-1, -1] and got.logprobs.tolist()[::2] == [0.0, 0.0]
    assert got.logprobs[1] == ops().token_logprobs(x, ints([4, 4, 4]), 0).logprobs[1]


def test_token_logprobs_refuses():
    x, t = torch.randn((3, 50), device="cuda"), ints([0, 1, 2])
    o = ops()
    for bad in (lambda: o.token_logprobs(x, t, 33), lambda: o.token_logprobs(x[:, :4], t, 5), lambda: o.token_logprobs(x, t, -1),
                lambda: o.token_logprobs(x, t.long(), 1), lambda: o.token_logprobs(x, t[:2], 1), lambda: o.token_logprobs(x.half(), t, 1),
                lambda: o.token_logprobs(x.t(), t, 1), lambda: o.token_logprobs(x.cpu(), t, 1), lambda: o.token_logprobs(x, t.cpu(), 1),
                lambda: o.token_logprobs(x, t, 1, blocks=3), lambda: o.token_logprobs(x, t, 1, blocks=32)):
        with pytest.raises(o.KernelError):
            bad()
    assert o.token_logprobs(x[:0], t[:0], 4).top_ids.shape == (0, 4)


# ------------------------------------------------------------------------------------------------ the step's tables
def same_layout(got, want):
    for name, a, b in zip(got._fields, got, want):
        assert (a is None) == (b is None), name
        if a is not None:
            assert a.dtype == torch.int32 and torch.equal(a.cpu(), b.cpu()), name


@pytest.mark.parametrize("q_lens,spare,tree", [([1], 0, True), ([1], 0, False), ([5, 0, 3, 1, 0], 7, True), ([0, 0], 4, True), ([3, 300, 40], 0, False),
                                               ([64, 33, 1, 32, 100], 31, True), ([1] * 300, 3, False), ([2] * 70, 0, True), ([1000], 24, True),
                                               ([], 3, False)])
@pytest.mark.parametrize("shape", ["mixed", "chain", "forest"])
def test_step_layout(q_lens, spare, tree, shape):
    g = random.Random(len(q_lens) + spare)
    S, N, ps = len(q_lens), sum(q_lens) + spare, 16
    ctx = [g.choice([0, 1, 15, 16, 17, 400]) for _ in q_lens]
    width = max([-(-(c + n) // ps) for c, n in zip(ctx, q_lens)] + [1]) + 1
    slots = g.sample(range(S + 5), S)
    rows = torch.tensor([[g.randrange(1, 9999) for _ in range(width + 2)] for _ in range(S + 5)], dtype=torch.int32)
    parents = torch.tensor([p for n in q_lens for p in make_parents(g, n, shape)] + [-1] * spare, dtype=torch.int32) if tree else None
    most = max(q_lens + [1])
    cpu = [torch.tensor(x, dtype=torch.int32) for x in (q_lens, ctx, slots)] + [rows]
    got = ops().step_layout(*[x.cuda() for x in cpu], ps, N, width, parents.cuda() if tree else None, most)
    want = ref_ops.step_layout(*cpu, ps, N, width, parents, most)
    same_layout(got, want)
    assert ops().read_status() == 0


def test_step_layout_raises_the_status_word():
    rows = torch.arange(1, 41, dtype=torch.int32).view(4, 10)

    def both(code, q, c, s, n, width=10, parents=None, most=0, rows=rows):
        cpu = [torch.tensor(x, dtype=torch.int32) for x in (q, c, s)] + [rows]
        up = None if parents is None else torch.tensor(parents, dtype=torch.int32)
        ref_ops.read_status()
        same_layout(ops().step_layout(*[x.cuda() for x in cpu], 4, n, width, None if up is None else up.cuda(), most),
                    ref_ops.step_layout(*cpu, 4, n, width, up, most))
        assert ops().read_status() == code and ref_ops.read_status() == code

    both(0, [3, 2], [1, 2], [0, 3], 6)
    both(32, [3, 9, 1], [1, 2, 0], [0, 3, 1], 6)              # more rows than there is room for
    both(32, [3, -2, 1], [1, 2, 0], [0, 3, 1], 6)
    both(8, [3, 2], [1, 2], [0, 4], 6)                        # a slot outside the slots
    both(8, [3, 2], [1, 2], [-1, 1], 6)
    both(16, [3, 2], [1, 39], [0, 1], 6)                      # a position outside the block table
    both(16, [3, 2], [1, 7], [0, 1], 6, width=2)
    both(16, [3, 2], [-1, 7], [0, 1], 6)
    both(64, [3, 2], [1, 2], [0, 1], 5, parents=[-1, 1, 0, -1, 0], most=4)         # hangs on itself
    both(64, [3, 2], [1, 2], [0, 1], 5, parents=[-1, 0, -5, -1, 0], most=4)
    both(64, [4, 2], [1, 2], [0, 1], 6, parents=[-1, 0, 1, 2, -1, 0], most=3)      # a tree of more rows than it may have
    both(4, [3, 2], [1, 2], [0, 1], 5, rows=-rows)


def test_step_layout_refuses():
    o, one, rows = ops(), ints([1]), ints([[1, 2]])
    ok = dict(q_lens=one, ctx_lens=one, slots=ints([0]), page_rows=rows, page_size=4, n_rows=1, width=2)
    o.step_layout(**ok)
    for kw in (dict(q_lens=one.cpu()), dict(q_lens=one.long()), dict(ctx_lens=ints([1, 2])), dict(slots=ints([[0]])), dict(page_rows=ints([1, 2])),
               dict(page_size=0), dict(width=0), dict(n_rows=-1), dict(parents=ints([-1]), tree_rows=0), dict(parents=ints([-1]), tree_rows=1025),
               dict(parents=ints([-1, 0]), tree_rows=4), dict(n_rows=1 << 22), dict(width=1 << 30, page_size=1 << 10)):
        with pytest.raises((o.KernelError, RuntimeError)):
            o.step_layout(**{**ok, **kw})
    assert o.read_status() == 0


# ------------------------------------------------------------------------------------------------ the accepted path
@pytest.mark.parametrize("q_lens,vocab", [([1], 5), ([2, 1, 6], 3), ([12, 0, 7, 33], 4), ([64, 40, 1, 200], 6), ([5] * 100, 2), ([1024], 2)])
@pytest.mark.parametrize("shape", ["mixed", "chain", "star", "forest"])
def test_accept_drafts(q_lens, vocab, shape):
    g = random.Random(sum(q_lens) + vocab)
    parents = [p for n in q_lens for p in make_parents(g, n, shape)]
    N, cu = len(parents), [0]
    for n in q_lens:
        cu.append(cu[-1] + n)
    tokens, choices = ([g.randrange(vocab) for _ in range(N)] for _ in range(2))
    step = SimpleNamespace(cu_q=ints(cu), ctx_lens=ints([g.randrange(100) for _ in q_lens]))
    args = (ints(choices), ints(tokens), ints(parents), step, max(q_lens))
    got, want = ops().accept_drafts(*args), ref_ops.accept_drafts(*args)
    for name, a, b in zip(got._fields, got, want):
        assert a.dtype == torch.int32 and torch.equal(a, b), name
    assert ops().read_status() == 0
    assert all(int(c) >= 1 for c, n in zip(got.counts, q_lens) if n)


def test_accept_drafts_raises_and_refuses():
    o = ops()
    step = SimpleNamespace(cu_q=ints([0, 3, 5]), ctx_lens=ints([4, 9]))
    a = [ints([7, 7, 7, 7, 7]), ints([7, 7, 7, 7, 7]), ints([-1, 0, 2, -1, 0])]
    got = o.accept_drafts(*a, step, 3)
    assert o.read_status() == 64 and got.counts.tolist() == [2, 2]
    got = o.accept_drafts(a[0], a[1], ints([-1, 0, 1, -1, 0]), step, 2)
    assert o.read_status() == 64 and got.counts.tolist() == [2, 2] and got.path.shape == (2, 2)
    bad = SimpleNamespace(cu_q=ints([0, 3, 9]), ctx_lens=step.ctx_lens)
    got = o.accept_drafts(a[0], a[1], ints([-1, 0, 1, -1, 0]), bad, 6)
    assert o.read_status() == 32 and got.counts.tolist() == [3, 0]
    for args in ((a[0][:4], a[1], a[2], step, 3), (a[0], a[1].long(), a[2], step, 3), (*a, step, 0), (*a, step, 2000),
                 (*a, SimpleNamespace(cu_q=step.cu_q, ctx_lens=ints([1])), 3), (a[0].cpu(), a[1], a[2], step, 3)):
        with pytest.raises(o.KernelError):
            o.accept_drafts(*args)


# ------------------------------------------------------------------------------------------------ accepted rows into the pages
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("planes,G,D,ps,strided", [(0, 2, 64, 16, False), (0, 2, 64, 16, True), (3, 8, 64, 64, False), (2, 1, 13, 5, False),
                                                   (1, 3, 20, 4, True), (0, 4, 128, 32, True), (2, 2, 320, 8, False)])
def test_commit_drafts(dtype, planes, G, D, ps, strided):
    g, t = random.Random(D), torch.Generator(device="cuda").manual_seed(D)
    q_lens, ctx = [5, 1, 9, 0, 30], [0, 15, 16, 3, 77]
    S, N, cu = len(q_lens), sum(q_lens), [0]
    for n in q_lens:
        cu.append(cu[-1] + n)
    ids = list(range(1, 400))
    g.shuffle(ids)
    table = [[ids.pop() for _ in range(-(-(c + n) // ps) + 1)] for c, n in zip(ctx, q_lens)]
    slots = [table[s][(ctx[s] + i) // ps] * ps + (ctx[s] + i) % ps for s in range(S) for i in range(q_lens[s])]
    slots[3] = -1                                              # a row without a place
    counts = [n if s == 0 else (n + 1) // 2 for s, n in enumerate(q_lens)]
    path = [sorted(g.sample(range(cu[s], cu[s + 1]), c)) + [-1] * (max(q_lens) - c) for s, c in enumerate(counts)]
    lead = (planes,) if planes else ()
    pages = torch.randn(lead + (400, 2, G, ps, D), generator=t, device="cuda").to(dtype)
    rows = torch.randn(lead + (N, 3 * G * D + 1), generator=t, device="cuda").to(dtype)
    k, v = rows[..., :G * D], rows[..., G * D:2 * G * D]
    if not strided:
        k, v = k.contiguous(), v.contiguous()
    step = SimpleNamespace(cu_q=ints(cu), kv_slots=ints(slots))
    want = pages.clone()
    ref_ops.commit_drafts(k, v, ints(path), ints(counts), step, want)
    ops().commit_drafts(k, v, ints(path), ints(counts), step, pages)
    assert torch.equal(pages, want)
    assert ops().read_status() == 0


def test_commit_drafts_raises_and_refuses():
    o = ops()
    pages, k = torch.zeros((6, 2, 1, 4, 8), dtype=BF16, device="cuda"), torch.ones((3, 8), dtype=BF16, device="cuda")
    step = SimpleNamespace(cu_q=ints([0, 3]), kv_slots=ints([4, 5, 24]))
    o.commit_drafts(k, k, ints([[0, 1, 2]]), ints([2]), step, pages)
    assert o.read_status() == 0 and int((pages != 0).sum()) == 32
    for path, counts, slots, code in (([[0, 1, 2]], [3], [4, 5, 24], 4), ([[0, 3, 1]], [2], [4, 5, 6], 32), ([[0, -1, 1]], [2], [4, 5, 6], 32),
                                      ([[0, 1, 2]], [4], [4, 5, 6], 32)):
        o.commit_drafts(k, k, ints(path), ints(counts), SimpleNamespace(cu_q=step.cu_q, kv_slots=ints(slots)), pages.clone())
        assert o.read_status() == code
    a = dict(k=k, v=k, path=ints([[0, 1, 2]]), counts=ints([2]), step=step, pages=pages)
    for kw in (dict(k=k.float()), dict(v=k[:2]), dict(pages=pages[0]), dict(pages=pages.float()), dict(path=ints([0, 1])), dict(counts=ints([1, 1])),
               dict(pages=torch.zeros((6, 1, 2, 4, 8), dtype=BF16, device="cuda")), dict(path=ints([[0]]).long()), dict(k=k.cpu())):
        with pytest.raises(o.KernelError):
            o.commit_drafts(**{**a, **kw})
    assert o.read_status() == 0


# ------------------------------------------------------------------------------------------------ streams and graphs
def test_operators_on_another_stream_and_in_graphs():
    """Two captured graphs of the same operators, replayed in turn and on two streams at once, keep nothing of one another."""
    o = ops()
    sets = []
    for seed, ctx in ((1, [300, 90]), (2, [40, 700])):
        q, k, v, step, cache, parents = make_tree_step([6, 9], ctx, 8, 2, 64, 16, BF16, seed)
        x, t = torch.randn((15, 9001), device="cuda"), ints([seed] * 15)
        up, tok = ints([p for ps in parents for p in ps]), ints([i % 3 for i in range(15)])

        def call(q=q, k=k, v=v, step=step, cache=cache, x=x, t=t, up=up, tok=tok):
            return [o.tree_attention(q, k, v, step, cache, 8, 2, 64, 0.125), *o.token_logprobs(x, t, 5), *o.accept_drafts(o.argmax(x) % 3, tok, up, step, 9)]
        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        sets.append((call, graph, out))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(20):
        for st, (_, graph, _) in zip(streams, sets):
            with torch.cuda.stream(st):
                graph.replay()
    torch.cuda.synchronize()
    for call, _, out in sets:
        with torch.cuda.stream(streams[0]):
            want = call()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b)
    assert o.read_status() == 0


# ------------------------------------------------------------------------------------------------ together, as a model runs them
@pytest.fixture(scope="module")
def tree_models(tmp_path_factory):
    from draft_configs import TREES_A, TREES_B
    from zig_ai_b200.config import config_from_dict
    from zig_ai_b200.weights import write_random_model
    out = {}
    for name, cfg in (("A", TREES_A), ("B", TREES_B)):
        out[name] = (str(tmp_path_factory.mktemp("trees") / name), cfg)
        write_random_model(config_from_dict(cfg), 5, out[name][0], matrix_std="fan_in")
    return out


@pytest.mark.parametrize("name,dtype", [("A", "float32"), ("A", "bfloat16"), ("B", "float32"), ("B", "bfloat16")])
def test_verified_trees_follow_the_plain_model(tree_models, name, dtype):
    """Generation by checked drafts: every token is the plain implementation's choice behind the tokens before it (in bfloat16 within what the
    model's rounding moves its logits, as for single tokens), most steps take more than one, and the cache's bookkeeping holds."""
    import plain_lfm2
    from draft_configs import speculate
    from zig_ai_b200.engine.runner import load_runner
    d, cfg = tree_models[name]
    V = cfg["vocab_size"]
    c, W = plain_lfm2.read_config(d), plain_lfm2.read_weights(d)
    g = random.Random(2)
    prompts = {f"r{i}": [g.randrange(V) for _ in range(n)] for i, n in enumerate([1, 19, 60])}
    truths = {}
    for rid, p in prompts.items():
        toks = list(p)
        for _ in range(30):
            toks.append(int(plain_lfm2.forward(c, W, toks)[-1].argmax()))
        truths[rid] = toks[len(p):]
    runner = load_runner(d, dtype, max_tokens=512, max_requests=4, page_size=16)
    got, steps = speculate(runner, prompts, 20, truths, g, V)
    if dtype == "float32":
        assert got == {r: t[:20] for r, t in truths.items()} and steps < 20
    for rid, out in got.items():
        logits = plain_lfm2.forward(c, W, prompts[rid] + out)
        for i, tok in enumerate(out):
            row = logits[len(prompts[rid]) + i - 1]
            assert float(row.max() - row[tok]) <= (1e-3 if dtype == "float32" else 8e-2 * float(row.abs().max()))


def test_layout_serves_the_kernels_that_are_there(tree_models):
    """A step laid out on the device from lengths runs through page writes and span attention as one packed on the host does."""
    from zig_ai_b200.cache.manager import CacheView
    from zig_ai_b200.engine.batch import pack_step
    o, H, G, D, ps = ops(), 4, 2, 64, 16
    g = torch.Generator(device="cuda").manual_seed(4)
    ctx, q_lens = [20, 0, 37], [5, 33, 10]
    table = [[3, 7, 0, 0], [5, 1, 9, 0], [2, 8, 6, 0]]
    host = pack_step(o, BF16, torch.device("cuda", 0), [(s, ctx[s], [0] * q_lens[s], [], s + 1) for s in range(3)], {0: table})
    rows = torch.zeros((5, 6), dtype=torch.int32, device="cuda")
    rows[[4, 1, 3], :4] = ints(table)
    lay = o.step_layout(ints(q_lens), ints(ctx), ints([4, 1, 3]), rows, ps, 48, 4)
    assert torch.equal(lay.positions, host.positions) and torch.equal(lay.seq_idx, host.seq_idx) and torch.equal(lay.cu_q[:4], host.cu_q)
    assert torch.equal(lay.block_tables[:3], host.block_tables[0]) and torch.equal(lay.ctx_lens[:3], host.ctx_lens)
    q, k, v = (torch.randn((48, n * D), generator=g, device="cuda").to(BF16) for n in (H, G, G))
    old = torch.randn((10, 2, G, ps, D), generator=g, device="cuda").to(BF16)
    outs = []
    for step, bt in ((host, host.block_tables[0]), (SimpleNamespace(**{**vars(host), "positions": lay.positions, "seq_idx": lay.seq_idx, "cu_q": lay.cu_q[:4],
                                                                       "ctx_lens": lay.ctx_lens[:3]}), lay.block_tables[:3])):
        view = CacheView(0, old.clone(), bt.contiguous(), ps)
        o.kv_write(k, v, step, view, G, D)
        outs.append((view.pages, o.paged_attention(q, step, view, H, G, D, 0.125)))
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])
    # a chain of drafts is a span: committing all of its rows writes the pages that kv_write writes
    pages, path = old.clone(), torch.full((3, 33), -1, dtype=torch.int32)
    for s, (a, n) in enumerate(zip([0, 5, 38], q_lens)):
        path[s, :n] = torch.arange(a, a + n)
    o.commit_drafts(k, v, path.cuda(), ints(q_lens), lay, pages)
    assert torch.equal(pages, outs[0][0])
    # and attention over a chain's masks is span attention
    chain = o.step_layout(ints(q_lens), ints(ctx), ints([4, 1, 3]), rows, ps, 48, 4, ints([i - 1 for n in q_lens for i in range(n)]), 33)
    assert torch.equal(chain.positions, lay.positions)
    step = SimpleNamespace(cu_q=chain.cu_q, ctx_lens=chain.ctx_lens, positions=chain.positions, tree_mask=chain.tree_mask, n_seqs=4, n_tokens=48, max_q_len=33)
    got = o.tree_attention(q, k, v, step, SimpleNamespace(pages=old, block_table=chain.block_tables, page_size=ps), H, G, D, 0.125)
    # (two kernels that each round the weights and the result to bfloat16: 2 (2^-8 sum p|v| + 2^-8 |o|), |v| < 6)
    assert float((got.float() - outs[0][1].float()).abs().max()) <= 4 * 2.0 ** -8 * float(v.float().abs().max())


# ------------------------------------------------------------------------------------------------ lengths near the type's end, padded steps
@pytest.mark.parametrize("dtype,impl", [(F32, None), (BF16, "general"), (BF16, "mma"), (BF16, "tcgen05")])
@pytest.mark.parametrize("ctx", [2 ** 31 - 1, 2 ** 31 - 100, 2 ** 30])
def test_lengths_beyond_the_block_table_raise_the_status_word(dtype, impl, ctx):
    """What lies beyond a block table's row has no page; the other requests' rows come out as they do without it."""
    o = ops()
    q, k, v, step, cache, _ = make_tree_step([3, 4], [40, 30], 8, 2, 64, 16, dtype, 3, poison=0.0)
    want = o.tree_attention(q, k, v, step, cache, 8, 2, 64, 0.125, impl=impl)
    assert o.read_status() == 0
    step.ctx_lens = ints([ctx, 30])
    got = o.tree_attention(q, k, v, step, cache, 8, 2, 64, 0.125, impl=impl)
    assert o.read_status() == 16
    tol = 2e-5 if dtype == F32 else 2.0 ** -6                  # (another share of the keys may go to other blocks: two roundings of weights and result)
    assert float((got[3:] - want[3:]).abs().max()) <= tol * float(v.float().abs().max())


def test_tables_of_lengths_near_the_types_end_raise_the_status_word():
    o, most = ops(), 2 ** 31 - 1
    rows = torch.arange(1, 41, dtype=torch.int32, device="cuda").view(4, 10)
    for ctx in (most, most - 1, 2 ** 30):
        lay = o.step_layout(ints([3, 2]), ints([ctx, 5]), ints([0, 1]), rows, 4, 6, 10, ints([-1, 0, 0, -1, 0, -1]), 3)
        assert o.read_status() == 16
        assert lay.kv_slots.tolist() == [-1, -1, -1, int(rows[1, 1]) * 4 + 1, int(rows[1, 1]) * 4 + 2, -1]
    one = ints([0, 0, 0, 0])
    for cu in ([2, most], [-3, 4], [most, most], [3, 1], [-most - 1, most]):
        step = SimpleNamespace(cu_q=ints(cu), ctx_lens=ints([7]), kv_slots=ints([4, 5, 6, 7]))
        got = o.accept_drafts(one, one, ints([-1, 0, 1, 2]), step, 4)
        assert got.counts.tolist() == [0] and got.path.tolist() == [[-1] * 4] and got.ctx_lens.tolist() == [7] and o.read_status() == 32
    pages, kv = torch.zeros((4, 2, 1, 4, 8), device="cuda"), torch.ones((4, 8), device="cuda")
    for first in (most, -1, -most - 1, 3):
        step = SimpleNamespace(cu_q=ints([first, 4]), ctx_lens=ints([7]), kv_slots=ints([4, 5, 6, 7]))
        o.commit_drafts(kv, kv, ints([[0, 1, 2]]), ints([3]), step, pages)
        assert o.read_status() == 32 and float(pages.sum()) == (16 if first == 3 else 0)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("spare", [1, 40, 200])
def test_rows_of_no_request_see_nothing(dtype, spare):
    """A step of fixed size: the rows behind the last tree are a span of no request, longer than any tree; they come out as zeros."""
    o, H, G, D, ps = ops(), 8, 2, 64, 16
    q, k, v, step, cache, parents = make_tree_step([5, 0, 9], [700, 3, 31], H, G, D, ps, dtype, 6)
    want = o.tree_attention(q, k, v, step, cache, H, G, D, 0.125)
    n, N = 14, 14 + spare
    wide = [torch.cat([x, torch.randn((spare, x.shape[1]), device="cuda").to(dtype)]) for x in (q, k, v)]
    lay = o.step_layout(ints([5, 0, 9]), step.ctx_lens, ints([0, 1, 2]), cache.block_table, ps, N, cache.block_table.shape[1],
                        ints([p for ps_ in parents for p in ps_] + [-1] * spare), 9)
    padded = SimpleNamespace(cu_q=lay.cu_q, ctx_lens=lay.ctx_lens, positions=lay.positions, tree_mask=lay.tree_mask, n_seqs=4, n_tokens=N, max_q_len=max(9, spare))
    got = o.tree_attention(*wide, padded, SimpleNamespace(pages=cache.pages, block_table=lay.block_tables, page_size=ps), H, G, D, 0.125)
    assert o.read_status() == 0 and not got[n:].any()
    assert torch.equal(lay.positions[:n], step.positions) and torch.equal(lay.tree_mask[:n], step.tree_mask)
    assert float((got[:n].float() - want.float()).abs().max()) <= (1e-5 if dtype == F32 else 2.0 ** -6) * float(v.float().abs().max())


def test_scores_beside_requests_that_are_served(tree_models):
    """A prompt scored while a decode step is on its way changes neither that step's requests nor its own log probabilities."""
    from zig_ai_b200.engine import Engine
    d, cfg = tree_models["A"]
    g = random.Random(12)
    prompts = [[g.randrange(cfg["vocab_size"]) for _ in range(n)] for n in (17, 5)]
    scored = [[g.randrange(cfg["vocab_size"]) for _ in range(n)] for n in (40, 2, 1)]

    def engine():
        return Engine(d, "float32", max_num_seqs=4, max_batched_tokens=32, max_model_len=128, page_size=16)
    alone = engine()
    want_out, want_score = alone.generate(prompts, max_new_tokens=12), alone.score(scored, top=2)
    eng = engine()
    from zig_ai_b200.sampling import SamplingParams
    ids = [eng.add_request(p, SamplingParams(temperature=0.0, max_new_tokens=12)) for p in prompts]
    done, n = {}, 0
    while eng.has_work():
        for r in eng.step():
            done[r.request_id] = r.output
        n += 1
        if n in (3, 5):
            got = eng.score(scored, top=2)
            for a, b in zip(got, want_score):
                assert [(e["token"], e["rank"], [t for t, _ in e["top"]]) for e in a] == [(e["token"], e["rank"], [t for t, _ in e["top"]]) for e in b]
                assert all(abs(x["logprob"] - y["logprob"]) < 1e-4 for x, y in zip(a, b))
    for r in eng.flush():
        done[r.request_id] = r.output
    assert [done[i] for i in ids] == want_out
    eng.runner.cache.check()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("ps", [8, 32, 128, 256])
def test_many_short_units(D, ps):
    """Shares of many units of one to four tiles, of one turn's pairs and of both turns' in any order, cached lengths at every side of a tile's border."""
    g, H, G = random.Random(ps + D), 8, 2
    for shape in ("mixed", "forest"):
        q_lens = [g.choice([0, 1, 2, 5, 31, 32, 33, 64, 65, 70, 128]) for _ in range(50)]
        ctx = [g.choice([0, 1, 63, 64, 65, 127, 128, 130, 200]) for _ in range(50)]
        q, k, v, step, cache, _ = make_tree_step(q_lens, ctx, H, G, D, ps, BF16, ps, shape, packed=shape == "mixed")
        got = ops().tree_attention(q, k, v, step, cache, H, G, D, D ** -0.5, impl="tcgen05")
        close(got, q, k, v, step, cache, H, G, D, D ** -0.5, None)
        for _ in range(5):
            assert torch.equal(ops().tree_attention(q, k, v, step, cache, H, G, D, D ** -0.5, impl="tcgen05"), got)
    assert ops().read_status() == 0


@pytest.mark.parametrize("D", [64, 128])
def test_what_is_not_finite_in_many_short_units(D):
    """Of 60 units in a row every third has a drafted value that is not finite: the rows that see it end so in that column, the others as without it."""
    g, H, G = random.Random(D), 8, 2
    q_lens, ctx = [g.choice([3, 9, 40, 70]) for _ in range(60)], [g.choice([0, 5, 64, 100]) for _ in range(60)]
    q, k, v, step, cache, parents = make_tree_step(q_lens, ctx, H, G, D, 16, BF16, 3)
    want = ops().tree_attention(q, k, v, step, cache, H, G, D, 0.125, impl="tcgen05")
    v = v.clone()
    sees, hit, cu = ref_ops._bits(step.tree_mask, 70), torch.zeros((sum(q_lens), H, D), dtype=torch.bool, device="cuda"), 0
    for s, n in enumerate(q_lens):
        if s % 3 == 0:
            row, head, col = g.randrange(n), g.randrange(G), g.randrange(D)
            v[cu + row, head * D + col] = g.choice([float("nan"), float("inf")])
            hit[cu:cu + n, head * (H // G):(head + 1) * (H // G), col] = sees[cu:cu + n, row][:, None]
        cu += n
    got = ops().tree_attention(q, k, v, step, cache, H, G, D, 0.125, impl="tcgen05").view(-1, H, D)
    assert not torch.isfinite(got[hit]).any() and torch.equal(got[~hit], want.view(-1, H, D)[~hit])
    assert ops().read_status() == 0


@pytest.mark.parametrize("impl", ["general", "mma", "tcgen05"])
@pytest.mark.parametrize("D,group,G", [(64, 3, 1), (128, 7, 2), (64, 1, 5), (128, 16, 1), (64, 40, 1)])
def test_other_head_layouts_and_columns_of_one_projection(impl, D, group, G):
    """q, k and v as columns of one product's rows; query heads that share a key/value head by threes, sevens and forties."""
    H = group * G
    q, k, v, step, cache, _ = make_tree_step([9, 1, 50], [70, 0, 300], H, G, D, 32, BF16, 4)
    rows = torch.cat([q, k, v], 1)
    q2, k2, v2 = rows[:, :H * D], rows[:, H * D:(H + G) * D], rows[:, (H + G) * D:]
    got = ops().tree_attention(q2, k2, v2, step, cache, H, G, D, D ** -0.5, impl=impl)
    close(got, q, k, v, step, cache, H, G, D, D ** -0.5, None)
    assert torch.equal(got, ops().tree_attention(q, k, v, step, cache, H, G, D, D ** -0.5, impl=impl)) and ops().read_status() == 0
