"""`Engine.score` on the CPU with the plain kernels: what it runs, and what it leaves of the engine that serves beside it."""
import pytest
import torch

import ref_ops
from draft_configs import TREES_A
from zig_ai_b200.config import config_from_dict
from zig_ai_b200.engine.engine import Engine
from zig_ai_b200.weights import write_random_model


@pytest.fixture(scope="module")
def model_dir(tmp_path_factory):
    d = str(tmp_path_factory.mktemp("score") / "m")
    write_random_model(config_from_dict(TREES_A), 5, d, matrix_std="fan_in")
    return d


def engine(d, portion=7):
    return Engine(d, "float32", max_num_seqs=2, max_batched_tokens=portion, max_model_len=64, page_size=4, device="cpu", ops=ref_ops)


def test_only_tokens_that_something_is_read_behind_are_run(model_dir):
    """The last token of a prompt has none behind it: it takes no row, and no step where it would be a portion's only one."""
    eng = engine(model_dir)
    for n, steps in ((1, 0), (2, 1), (7, 1), (8, 1), (9, 2), (15, 2), (16, 3)):
        before = eng.runner.steps, eng.runner.tokens_run
        entries, = eng.score([[i % 61 for i in range(n)]])
        assert len(entries) == n - 1
        assert (eng.runner.steps - before[0], eng.runner.tokens_run - before[1]) == (steps, n - 1)
    assert not eng.runner.processed
    eng.runner.cache.check()


def test_scored_portions_make_no_step_graphs(model_dir):
    """A graph of a scored portion would keep logits of every row (2048 x 65 536 in 32 bits: half a GB) and push out those of served steps."""
    eng = engine(model_dir)

    class Graphs:
        asked = 0

        def bucket(self, n):
            return None

        def run(self, spans, tables):
            Graphs.asked += 1

    want = eng.score([list(range(20))] * 2, top=2)
    r = eng.runner
    r.use_graphs, r.graphs, r.shape_graphs = True, Graphs(), Graphs()
    assert eng.score([list(range(20))] * 2, top=2) == want and Graphs.asked == 0
    r.add_request("a")
    r.step([("a", [1, 2, 3], [2])])
    assert Graphs.asked == 1
