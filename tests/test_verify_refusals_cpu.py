"""What a refused `ModelRunner.verify` leaves behind (nothing), and trees through layers that see a window of positions, on the CPU with the
plain kernels."""
import random

import pytest
import torch

import ref_ops
from draft_configs import TREES_A, draft, speculate
from window_configs import WINDOWED, windowed_layers
from zig_ai_b200.config import config_from_dict
from zig_ai_b200.engine.runner import StepError, load_runner
from zig_ai_b200.weights import write_random_model

V = TREES_A["vocab_size"]


@pytest.fixture(scope="module")
def dirs(tmp_path_factory):
    out = {}
    with windowed_layers(6):
        for name, cfg in (("full", TREES_A), ("window", {**TREES_A, "architectures": [WINDOWED]})):
            out[name] = str(tmp_path_factory.mktemp("refused") / name)
            write_random_model(config_from_dict(cfg), 5, out[name], matrix_std="fan_in")
        yield out


def runner(d, max_tokens=512):
    return load_runner(d, "float32", max_tokens=max_tokens, max_requests=4, page_size=4, device="cpu", ops=ref_ops)


def greedy(d, prompt, n):
    r = runner(d)
    r.add_request("a")
    out, toks = [], list(prompt)
    for _ in range(n):
        toks = [int(r.step([("a", toks, [len(toks) - 1])])[0].argmax())]
        out += toks
    return out


class Refused(Exception):
    pass


def raises(logits):
    raise Refused("no choice")


REFUSALS = {"shape": (lambda x: x.argmax(-1)[:1], StepError), "raise": (raises, Refused)}


def holds(r, rid, n):
    assert r.processed[rid] == n and r.cache.requests[rid].num_tokens == n
    r.cache.check()


@pytest.mark.parametrize("how", REFUSALS)
@pytest.mark.parametrize("name", ["full", "window"])
def test_a_refused_choice_gives_its_positions_back(dirs, name, how):
    """After it the request goes on as if it had not been: by a single token, by a tree of fewer rows, by one of more."""
    choose, error = REFUSALS[how]
    prompt = [5, 9, 11, 3, 2, 60, 7, 7, 1, 30]
    want = greedy(dirs[name], prompt, 14)
    for then in ("step", "shorter", "longer"):
        r = runner(dirs[name])
        r.add_request("a")
        r.step([("a", prompt[:-1], [])])
        for rows in (3, 12, 9):
            with pytest.raises(error):
                r.verify([("a", [prompt[-1]] + [0] * (rows - 1), [-1] + [0] * (rows - 1))], choose)
            holds(r, "a", 9)
        if then == "step":
            got = [int(r.step([("a", prompt[-1:], [0])])[0].argmax())]
        else:
            tokens = [prompt[-1]] + want[:2] + ([0] * 13 if then == "longer" else [])
            got = r.verify([("a", tokens, list(range(-1, len(tokens) - 1)))])[0]
        holds(r, "a", 9 + len(got))
        while len(got) < 14:
            got += r.verify([("a", [got[-1], 4], [-1, 0])])[0]
        assert got[:14] == want
        r.end_request("a")
        r.cache.check()
    assert ref_ops.read_status() == 0


def test_a_step_without_room_gives_every_requests_positions_back(dirs):
    """A refusal of the layout, the forward pass or a later operator is one of the whole step."""
    r = runner(dirs["full"])
    for rid in "ab":
        r.add_request(rid)
        r.step([(rid, [1, 2, 3], [])])

    class Ops:
        def __getattr__(self, name):
            return getattr(ref_ops, name)

    for name in ("step_layout", "tree_attention", "accept_drafts", "commit_drafts"):
        ops = Ops()
        setattr(ops, name, lambda *a, **k: raises(None))
        r.ops = ops
        with pytest.raises(Refused):
            r.verify([("a", [4, 5], [-1, 0]), ("b", [6, 5, 4], [-1, 0, 0])])
        for rid in "ab":
            holds(r, rid, 3)
    r.ops = ref_ops
    assert all(r.verify([("a", [4], [-1]), ("b", [6], [-1])]))


def test_trees_in_windowed_layers_give_the_tokens_of_single_steps(dirs):
    """Rejected drafts across the borders of pages that the window has left or is about to leave, refused choices between the steps."""
    g = random.Random(11)
    prompts = {f"r{i}": [g.randrange(V) for _ in range(n)] for i, n in enumerate([1, 7, 16])}
    want = {k: greedy(dirs["window"], p, 40) for k, p in prompts.items()}
    got, steps = speculate(runner(dirs["window"]), prompts, 30, want, g, V, most=14)
    assert got == {k: t[:30] for k, t in want.items()} and steps < 30
    r = runner(dirs["window"])
    r.add_request("a")
    r.step([("a", prompts["r2"][:-1], [])])
    out, last = [], prompts["r2"][-1]
    while len(out) < 24:
        tokens, parents = draft(g, [last] + want["r2"][len(out):], g.randint(1, 13), V)
        with pytest.raises(Refused):
            more = g.randrange(9)                           # (a refused tree larger than the next one, or the same)
            r.verify([("a", tokens + [0] * more, parents + [0] * more)], raises)
        holds(r, "a", 15 + len(out))
        out += r.verify([("a", tokens, parents)])[0]
        last = out[-1]
    assert out == want["r2"][:len(out)]
    assert ref_ops.read_status() == 0


def test_a_raised_status_word_is_read_before_the_counts_are_used(dirs):
    """A step whose kernels raised the status word accepts nothing: lengths stay, whatever the counts say, and the next step is not blamed."""
    for counts in (None, 99, -3):
        r = runner(dirs["full"])
        for rid in "ab":
            r.add_request(rid)
            r.step([(rid, [1, 2, 3], [])])

        class Ops:
            def __getattr__(self, name):
                return getattr(ref_ops, name)

            def accept_drafts(self, *a):
                out = ref_ops.accept_drafts(*a)
                ref_ops._raise(64)
                return out if counts is None else out._replace(counts=torch.full_like(out.counts, counts))

            def commit_drafts(self, *a):
                pass

        r.ops = Ops()
        steps = r.steps
        with pytest.raises(StepError, match=f"step {steps}: .*status 64.*void"):
            r.verify([("a", [4, 5], [-1, 0]), ("b", [6, 5, 4], [-1, 0, 0])])
        for rid in "ab":
            holds(r, rid, 3)
        r.ops = ref_ops
        assert ref_ops.read_status() == 0
        assert all(r.verify([("a", [4], [-1]), ("b", [6], [-1])]))
