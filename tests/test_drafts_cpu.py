"""Steps that check drafted tokens, on the CPU: `ModelRunner.verify` and `Engine.score` with the plain kernels against single tokens one after
the other, the cache's bookkeeping, what is refused, and the C entry points' own refusals (they launch nothing then)."""
import ctypes
import random

import pytest
import torch

import plain_lfm2
import ref_ops
from draft_configs import TREES_A, draft, speculate
from zig_ai_b200.config import config_from_dict
from zig_ai_b200.engine.engine import Engine
from zig_ai_b200.engine.runner import StepError, load_runner
from zig_ai_b200.weights import write_random_model


@pytest.fixture(scope="module")
def model_dir(tmp_path_factory):
    d = str(tmp_path_factory.mktemp("trees") / "m")
    write_random_model(config_from_dict(TREES_A), 5, d, matrix_std="fan_in")
    return d


def runner(model_dir, max_tokens=512):
    return load_runner(model_dir, "float32", max_tokens=max_tokens, max_requests=4, page_size=4, device="cpu", ops=ref_ops)


def greedy(model_dir, prompt, n):
    r = runner(model_dir)
    r.add_request("a")
    out, toks = [], list(prompt)
    for _ in range(n):
        logits = r.step([("a", toks, [len(toks) - 1])])
        toks = [int(logits[0].argmax())]
        out += toks
    return out


def test_verified_trees_give_the_tokens_of_single_steps(model_dir):
    g = random.Random(3)
    prompts = {f"r{i}": [g.randrange(61) for _ in range(n)] for i, n in enumerate([1, 7, 16])}
    want = {k: greedy(model_dir, p, 40) for k, p in prompts.items()}
    got, steps = speculate(runner(model_dir), prompts, 24, want, g, 61)
    assert got == {k: t[:24] for k, t in want.items()}
    assert steps < 24 and ref_ops.read_status() == 0


def test_verify_then_single_steps_go_on_from_the_accepted_tokens(model_dir):
    p, want = [5, 9, 11], None
    want = greedy(model_dir, p, 12)
    r = runner(model_dir)
    r.add_request("a")
    r.step([("a", p[:2], [])])
    toks = r.verify([("a", [11, want[0], 3, want[1], want[2]], [-1, 0, 0, 1, 3])])[0]
    assert toks == want[:4] and r.processed["a"] == 2 + 4 and r.cache.requests["a"].num_tokens == 6
    for w in want[4:]:
        toks = [int(r.step([("a", [toks[-1]], [0])])[0].argmax())]
        assert toks == [w]


def test_verify_refuses(model_dir, tiny_models):
    r = runner(model_dir, max_tokens=16)
    r.add_request("a")
    for tokens, parents in (([1, 2], [-1]), ([1, 2], [-1, 1]), ([1, 2], [0, 0]), ([1, 2, 3], [-1, 0, -1]), ([], []), ([1, 99], [-1, 0]), ([1], [-2])):
        with pytest.raises(StepError):
            r.verify([("a", tokens, parents)])
    with pytest.raises(StepError):
        r.verify([("b", [1], [-1])])
    with pytest.raises(Exception, match="pages"):
        r.verify([("a", list(range(17)), [-1] + [0] * 16)])
    assert r.processed["a"] == 0 and r.verify([("a", [1], [-1])])
    other = load_runner(tiny_models["A"], "float32", max_tokens=64, max_requests=2, page_size=8, device="cpu", ops=ref_ops)
    other.add_request("a")
    assert not other.takes_trees()
    with pytest.raises(StepError, match="layers"):
        other.verify([("a", [1], [-1])])


def test_settle_keeps_pages_and_refuses_more_than_is_reserved(model_dir):
    r = runner(model_dir)
    r.add_request("a")
    c = r.cache
    c.reserve("a", 11)
    held = dict(c.requests["a"].tables)
    c.settle("a", 5)
    assert c.requests["a"].num_tokens == 5 and c.requests["a"].tables == held
    c.reserve("a", 12)
    with pytest.raises(ValueError):
        c.settle("a", 13)
    with pytest.raises(ValueError):
        c.settle("a", -1)
    r.end_request("a")
    c.check()


def test_a_draft_is_a_tree():
    g = random.Random(1)
    for n in range(1, 30):
        tokens, parents = draft(g, [1, 2, 3, 4], n, 10)
        assert len(tokens) == n and parents[0] == -1 and all(0 <= parents[i] < i for i in range(1, n))


def test_scores_are_the_plain_models_log_probabilities(model_dir):
    g = random.Random(8)
    prompts = [[g.randrange(61) for _ in range(n)] for n in (1, 2, 30, 9)]
    eng = Engine(model_dir, "float32", max_num_seqs=2, max_batched_tokens=7, max_model_len=64, page_size=4, device="cpu", ops=ref_ops)
    got = eng.score(prompts, top=3)
    c, W = plain_lfm2.read_config(model_dir), plain_lfm2.read_weights(model_dir)
    for p, entries in zip(prompts, got):
        assert len(entries) == len(p) - 1
        lp = torch.log_softmax(plain_lfm2.forward(c, W, p), -1)
        for i, e in enumerate(entries):
            assert e["token"] == p[i + 1] and abs(e["logprob"] - float(lp[i, p[i + 1]])) < 1e-3
            assert e["rank"] == int((lp[i] > lp[i, p[i + 1]]).sum()) or abs(float(lp[i].sort().values.diff().abs().min())) < 1e-3
            assert abs(e["entropy"] + float((lp[i].exp() * lp[i]).sum())) < 1e-3 and len(e["top"]) == 3
            assert e["top"][0][1] >= e["top"][1][1] >= e["top"][2][1]
    assert not eng.runner.processed
    eng.runner.cache.check()
    with pytest.raises(ValueError):
        eng.score([[]])
    with pytest.raises(ValueError):
        eng.score([[1] * 65])


def c_entry(lib, name):
    from zig_ai_b200.kernels import build, ops
    f = getattr(build.load(lib), name)
    f.argtypes, f.restype = ops._SIGNATURES[lib][name], ctypes.c_int
    return f


def test_c_entry_points_refuse_sizes_before_they_launch():
    """Each call has one size or type out of range; none reaches a device (there need be none)."""
    p = 1 << 20                                               # (an address that nothing looks at)
    layout = dict(S=2, N=8, width=4, row_width=4, n_slots=3, page_size=16, tree_rows=4, words=1)
    f = c_entry("drafts", "zai_step_layout")
    for kw in (dict(S=-1), dict(S=8193), dict(N=-1), dict(N=1 << 22), dict(width=0), dict(row_width=0), dict(n_slots=0), dict(page_size=0),
               dict(tree_rows=1025, words=33), dict(tree_rows=40), dict(words=33), dict(width=1 << 20, page_size=1 << 12)):
        a = {**layout, **kw}
        assert f(*[p] * 12, *a.values(), p, None) == -2, kw
    f = c_entry("drafts", "zai_accept_drafts")
    for S, N, most in ((0, 4, 4), (2, -1, 4), (2, 4, 0), (2, 4, 1025)):
        assert f(*[p] * 9, S, N, most, p, None) == -2
    f = c_entry("drafts", "zai_commit_drafts")
    sizes = dict(dtype=1, S=2, N=4, most=3, planes=1, kv_heads=2, head_dim=64, page_size=16, num_pages=9)
    for kw in (dict(S=0), dict(N=-1), dict(most=0), dict(planes=0), dict(planes=65536), dict(kv_heads=0), dict(head_dim=0), dict(page_size=0), dict(num_pages=0)):
        assert f(p, p, p, 0, 0, 128, 128, p, p, p, p, *{**sizes, **kw}.values(), p, None) == -2, kw
    assert f(p, p, p, 0, 0, 128, 128, p, p, p, p, *{**sizes, "dtype": 7}.values(), p, None) == -1
    f = c_entry("logprobs", "zai_token_logprobs")
    sizes = dict(R=2, V=100, top=5, blocks=1)
    for kw in (dict(R=0), dict(V=0), dict(top=-1), dict(top=33), dict(V=4), dict(blocks=3), dict(blocks=32), dict(blocks=-1)):
        assert f(p, p, p, p, p, p, 0, 100, p, *{**sizes, **kw}.values(), 148, p, None) == -2, kw
    assert f(p, p, p, p, p, p, 5, 100, p, 2, 100, 5, 1, 148, p, None) == -1
    sizes = dict(words=1, S=2, N=4, pairs=16, tiles=2, splits=1, page_size=16, num_pages=9, H=4, G=2, D=64)
    f = c_entry("tree_attention", "zai_tree_attention_mma")
    def mma(q=p, ks=128, **kw):
        return f(p, q, 256, p, ks, p, 128, p, p, 4, p, p, p, p, *{**sizes, **kw}.values(), 0.1, 0, p, None)
    for kw in (dict(words=0), dict(S=0), dict(N=0), dict(pairs=48), dict(tiles=0), dict(splits=0), dict(splits=17), dict(page_size=0), dict(num_pages=0),
               dict(H=5), dict(G=0), dict(D=80), dict(q=p + 2), dict(ks=130)):
        assert mma(**kw) == -2, kw
    f = c_entry("tree_attention", "zai_tree_attention_general")
    del sizes["pairs"]
    def general(dtype=0, **kw):
        return f(p, p, 256, p, 128, p, 128, p, dtype, p, 4, p, p, p, p, *{**sizes, **kw}.values(), 0.1, 0, p, None)
    for kw in (dict(words=0), dict(S=0), dict(N=0), dict(tiles=0), dict(splits=0), dict(splits=17), dict(H=5), dict(G=0), dict(D=0), dict(D=513)):
        assert general(**kw) == -2, kw
    assert general(dtype=3) == -1
    f = c_entry("tree_attention_tc", "zai_tree_attention_tc")
    sizes = dict(words=1, S=2, N=4, blocks=148, page_size=16, num_pages=9, H=4, G=2, D=64)
    def tc(q=p, qs=256, **kw):
        return f(p, q, qs, p, 128, p, 128, p, p, 4, p, p, p, *{**sizes, **kw}.values(), 0.1, p, p, None)
    for kw in (dict(words=0), dict(S=0), dict(N=0), dict(blocks=0), dict(page_size=12), dict(page_size=4), dict(num_pages=0), dict(H=5), dict(G=0), dict(D=96),
               dict(q=p + 8), dict(qs=260)):
        assert tc(**kw) == -2, kw


def test_wrappers_refuse_tensors_off_the_device():
    from types import SimpleNamespace
    from zig_ai_b200.kernels import ops
    i = torch.zeros(3, dtype=torch.int32)
    step = SimpleNamespace(cu_q=torch.zeros(4, dtype=torch.int32), ctx_lens=i, positions=i, tree_mask=i.view(3, 1), kv_slots=i, n_seqs=3, n_tokens=3, max_q_len=1)
    x = torch.zeros(3, 64)
    cache = SimpleNamespace(pages=torch.zeros(2, 2, 1, 4, 64), block_table=i.view(3, 1), page_size=4)
    for call in (lambda: ops.tree_attention(x, x, x, step, cache, 1, 1, 64, 1.0), lambda: ops.token_logprobs(x, i), lambda: ops.step_layout(i, i, i, i.view(3, 1), 4, 3, 1),
                 lambda: ops.accept_drafts(i, i, i, step, 2), lambda: ops.commit_drafts(x, x, i.view(3, 1), i, step, cache.pages)):
        with pytest.raises(ops.KernelError):
            call()


def test_a_refused_score_or_choice_leaves_nothing_behind(model_dir):
    eng = Engine(model_dir, "float32", max_num_seqs=2, max_batched_tokens=7, max_model_len=64, page_size=4, device="cpu", ops=ref_ops)
    for prompts, top in (([[1, 2, 61]], 0), ([[1] * 9 + [-1]], 0), ([[1, 2]], 33), ([[1, 2]], -1), ([[1, 1 << 40]], 0)):
        with pytest.raises(ValueError):
            eng.score(prompts, top=top)
    runner = eng.runner
    assert not runner.processed
    runner.add_request("a")
    runner.step([("a", [1, 2, 3], [2])])
    for choose in (lambda x: x.argmax(-1)[:1], lambda x: x.argmax(-1, keepdim=True)):
        with pytest.raises(ValueError):
            runner.verify([("a", [4, 5], [-1, 0])], choose)
    assert runner.processed["a"] == 3
    assert len(runner.verify([("a", [4, 5], [-1, 0])])[0]) in (1, 2)
    runner.end_request("a")
    runner.cache.check()
