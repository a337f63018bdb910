"""Tree attention under windows whose keys are shared by several blocks, against 64 bits, and trees of drafted tokens through layers
that see a window of positions."""
import random

import pytest
import torch

from test_gpu_drafts import BF16, F32, close, make_tree_step, ops
from window_configs import WINDOWED, windowed_layers

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,impl", [(F32, None), (BF16, "general"), (BF16, "mma")])
@pytest.mark.parametrize("splits", [1, 2, 4, 8, 16])
@pytest.mark.parametrize("D,group,n,ps", [(64, 2, 5, 16), (64, 4, 14, 64), (128, 4, 30, 16), (96, 1, 9, 8), (32, 8, 40, 32)])
def test_windows_by_every_split(dtype, impl, splits, D, group, n, ps):
    """Blocks that begin behind the window's first tile, windows of fewer tiles than there are blocks, windows longer than all there is, spans
    whose rows see different first keys."""
    for window in (1, 3, 64, 333, 650, 5000):
        for shape in ("chain", "forest"):
            q, k, v, step, cache, _ = make_tree_step([n, 1, n, 2], [700, 3, 129, 1000], 2 * group, 2, D, ps, dtype, 11, shape)
            got = ops().tree_attention(q, k, v, step, cache, 2 * group, 2, D, D ** -0.5, window, impl=impl, splits=splits)
            close(got, q, k, v, step, cache, 2 * group, 2, D, D ** -0.5, window)
    assert ops().read_status() == 0


@pytest.mark.parametrize("dtype,impl", [(F32, None), (BF16, "general"), (BF16, "mma")])
@pytest.mark.parametrize("splits", [2, 4, 16])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_what_is_not_finite_behind_a_window_shared_by_blocks(dtype, impl, splits, bad):
    """Values at the edges of the rows' windows: they reach the rows that see them and no others."""
    H, G, D, ps, window = 4, 2, 64, 16, 300
    q, k, v, step, cache, _ = make_tree_step([40], [700], H, G, D, ps, dtype, 6, "chain")
    clean = ops().tree_attention(q, k, v, step, cache, H, G, D, 0.125, window, impl=impl, splits=splits)
    for at in (401, 415, 439, 440):                            # the row at position 700 + i sees keys from 401 + i on
        table = cache.block_table[0].tolist()
        place = cache.pages[table[at // ps], 1, :, at % ps]
        kept = place.clone()
        place.fill_(bad)
        got = ops().tree_attention(q, k, v, step, cache, H, G, D, 0.125, window, impl=impl, splits=splits)
        place.copy_(kept)
        sees = min(at - 401 + 1, 40)
        assert torch.equal(got[sees:], clean[sees:]) and not torch.isfinite(got[:sees]).any()
    assert ops().read_status() == 0


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("window", [20, 100])
def test_verified_trees_in_windowed_layers(tmp_path, dtype, window):
    """In 32 bits the tokens of single steps; in bfloat16 choices that are within its rounding of the 32-bit model's."""
    from draft_configs import TREES_B, speculate
    from zig_ai_b200.config import config_from_dict
    from zig_ai_b200.engine.runner import load_runner
    from zig_ai_b200.weights import write_random_model
    V, d = TREES_B["vocab_size"], str(tmp_path / "m")
    g = random.Random(2)
    prompts = {f"r{i}": [g.randrange(V) for _ in range(n)] for i, n in enumerate([1, 45, 130])}
    with windowed_layers(window):
        write_random_model(config_from_dict({**TREES_B, "architectures": [WINDOWED]}), 5, d, matrix_std="fan_in")
        exact = load_runner(d, "float32", max_tokens=1024, max_requests=4, page_size=16)
        truths = {}
        for rid, p in prompts.items():
            exact.add_request(rid)
            toks, out = p, []
            for _ in range(45):
                toks = [int(exact.step([(rid, toks, [len(toks) - 1])])[0].argmax())]
                out += toks
            exact.end_request(rid)
            truths[rid] = out
        runner = load_runner(d, dtype, max_tokens=1024, max_requests=4, page_size=16)
        got, steps = speculate(runner, prompts, 32, truths, g, V, most=12)
        if dtype == "float32":
            assert got == {r: t[:32] for r, t in truths.items()} and steps < 32
        for rid, out in got.items():
            exact.add_request(rid)
            toks = prompts[rid] + out
            logits = exact.step([(rid, toks, list(range(len(toks))))])
            exact.end_request(rid)
            for i, tok in enumerate(out):
                row = logits[len(prompts[rid]) + i - 1]
                assert float(row.max() - row[tok]) <= (1e-3 if dtype == "float32" else 8e-2 * float(row.abs().max()))
        # a refused choice, then a tree of fewer rows, then single tokens
        runner.add_request("a")
        p = prompts["r2"]
        runner.step([("a", p[:-1], [])])
        with pytest.raises(ValueError):
            runner.verify([("a", [p[-1]] + [0] * 40, [-1] + [0] * 40)], lambda x: x.argmax(-1)[:1])
        out = runner.verify([("a", [p[-1], truths["r2"][0]], [-1, 0])])[0]
        while len(out) < 30:
            out.append(int(runner.step([("a", [out[-1]], [0])])[0].argmax()))
        assert dtype != "float32" or out[:30] == truths["r2"][:30]
        runner.end_request("a")
        runner.cache.check()
    assert runner.ops.read_status() == 0


@pytest.mark.parametrize("D,dtype,impl", [(64, F32, None), (64, BF16, "general"), (64, BF16, "mma"), (64, BF16, "tcgen05"), (128, BF16, "tcgen05")])
def test_the_same_call_gives_the_same_bits(D, dtype, impl):
    """No order of atomics, no workspace that a call before has left something in."""
    H, G = 8, 2
    q, k, v, step, cache, _ = make_tree_step([24, 9, 60, 1, 33], [900, 0, 5000, 70, 2222], H, G, D, 64, dtype, 3)
    other = make_tree_step([7, 64], [300, 8000], H, G, D, 64, dtype, 4)
    want = ops().tree_attention(q, k, v, step, cache, H, G, D, D ** -0.5, impl=impl)
    for _ in range(30):
        ops().tree_attention(*other[:5], H, G, D, D ** -0.5, impl=impl)
        assert torch.equal(ops().tree_attention(q, k, v, step, cache, H, G, D, D ** -0.5, impl=impl), want)
    assert ops().read_status() == 0


@pytest.mark.parametrize("dtype,impl", [(F32, None), (BF16, "general"), (BF16, "mma"), (BF16, "tcgen05")])
@pytest.mark.parametrize("cu", [[0, 5, 7], [1, 5, 8], [0, 6, 4, 8], [0, 0], [0, 8, 7]])
def test_rows_of_no_span_raise_the_status_word(dtype, impl, cu):
    """A row that no span holds has no output, and a span of fewer than no rows is none: the step is void, and says so."""
    q, k, v, step, cache, _ = make_tree_step([5, 3], [20, 130], 4, 2, 64, 16, dtype, 9)
    S = len(cu) - 1
    step.cu_q, step.n_seqs, step.max_q_len = torch.tensor(cu, dtype=torch.int32, device="cuda"), S, 8
    step.ctx_lens, cache.block_table = step.ctx_lens[[0, 1, 1][:S]].contiguous(), cache.block_table[[0, 1, 1][:S]].contiguous()
    ops().tree_attention(q, k, v, step, cache, 4, 2, 64, 0.125, impl=impl)
    assert ops().read_status() == 32


@pytest.mark.parametrize("S", [1, 31, 32, 33, 64, 65, 100])
@pytest.mark.parametrize("dtype,impl", [(F32, None), (BF16, "mma"), (BF16, "tcgen05")])
def test_spans_without_rows_at_both_ends_are_no_fault(S, dtype, impl):
    """Rows in one span among many: the others hold none, and every row is in a span."""
    for at in {0, S // 2, S - 1}:
        q, k, v, step, cache, _ = make_tree_step([0] * at + [7] + [0] * (S - 1 - at), [33] * S, 4, 2, 64, 16, dtype, 9)
        got = ops().tree_attention(q, k, v, step, cache, 4, 2, 64, 0.125, impl=impl)
        assert ops().read_status() == 0
        close(got, q, k, v, step, cache, 4, 2, 64, 0.125, None)


def test_sizes_beyond_32_bits_keep_their_meaning():
    """A window of 2^32 + 5 positions is no window of five; tables are not laid out for a page size or a row count that wraps."""
    o = ops()
    for dtype, impl in ((F32, None), (BF16, "mma")):
        q, k, v, step, cache, _ = make_tree_step([5, 3], [20, 130], 4, 2, 64, 16, dtype, 9)
        want = o.tree_attention(q, k, v, step, cache, 4, 2, 64, 0.125, 0x7fffffff, impl=impl, splits=2)
        close(want, q, k, v, step, cache, 4, 2, 64, 0.125, None)
        for window in (1 << 31, (1 << 32) + 5, 1 << 40):
            assert torch.equal(o.tree_attention(q, k, v, step, cache, 4, 2, 64, 0.125, window, impl=impl, splits=2), want)
    one, rows = torch.ones(1, dtype=torch.int32, device="cuda"), torch.ones((2, 3), dtype=torch.int32, device="cuda")
    for kw in (dict(page_size=(1 << 32) + 4), dict(n_rows=1 << 32), dict(width=(1 << 32) + 1)):
        with pytest.raises(o.KernelError):
            o.step_layout(**{**dict(q_lens=one, ctx_lens=one, slots=one, page_rows=rows, page_size=4, n_rows=1, width=2), **kw})
    assert o.read_status() == 0


def test_the_largest_trees_of_the_tcgen05_kernel():
    """As many rows as the kernel says it takes, and one more: that goes to another kernel, or is refused."""
    o = ops()
    most = o._tree_kernel_takes("tc_rows")
    for n in (most, most + 1):
        q, k, v, step, cache, _ = make_tree_step([n, 2], [5000, 40], 4, 2, 64, 64, BF16, 9)
        close(o.tree_attention(q, k, v, step, cache, 4, 2, 64, 0.125), q, k, v, step, cache, 4, 2, 64, 0.125, None)
        if n == most:
            close(o.tree_attention(q, k, v, step, cache, 4, 2, 64, 0.125, impl="tcgen05"), q, k, v, step, cache, 4, 2, 64, 0.125, None)
            continue
        with pytest.raises(o.KernelError, match="128 rows"):
            o.tree_attention(q, k, v, step, cache, 4, 2, 64, 0.125, impl="tcgen05")
    assert o.read_status() == 0
