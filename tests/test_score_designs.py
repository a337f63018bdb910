"""`Engine.score` through every design: scored prompts cut into portions, whose states go through the requests' slots, against the plain
implementations; on the CPU with the plain kernels, on the GPU with the kernels in both types."""
import json
import os
import random

import pytest
import torch

import lolivik_configs
import pikasun_configs
import pirozen_configs
import plain_lfm2
import plain_lolivik
import plain_pikasun
import plain_pirozen
import plain_sogenex
import plain_vunolorn
import plain_zikevik
import ref_ops
import sogenex_configs
import tiny_configs
import vunolorn_configs
import zikevik_configs
from zig_ai_b200.config import config_from_dict
from zig_ai_b200.engine.engine import Engine
from zig_ai_b200.sampling.sampler import SamplingParams
from zig_ai_b200.weights import write_random_model
from zig_ai_b200.weights.safetensors_io import SafetensorsFile

DESIGNS = {"lfm2": (tiny_configs.TINY, plain_lfm2), "vunolorn": (vunolorn_configs.ALL, plain_vunolorn), "zikevik": (zikevik_configs.ALL, plain_zikevik),
           "sogenex": (sogenex_configs.ALL, plain_sogenex), "pirozen": (pirozen_configs.ALL, plain_pirozen),
           "pikasun": (pikasun_configs.ALL, plain_pikasun), "lolivik": (lolivik_configs.ALL, plain_lolivik)}
WRITERS = {"pirozen": pirozen_configs.write_model, "sogenex": sogenex_configs.write_model}


@pytest.fixture(scope="module")
def model(tmp_path_factory):
    made = {}

    def get(design, size):
        if (design, size) not in made:
            cfg, seed = DESIGNS[design][0][size]
            d = str(tmp_path_factory.mktemp("score") / design)
            if design in WRITERS:
                WRITERS[design](cfg, seed, d)
            else:
                write_random_model(config_from_dict(cfg), seed, d, matrix_std="fan_in")
            made[design, size] = d
        return made[design, size]
    return get


def plain(design, d, tokens):
    P = DESIGNS[design][1]
    if hasattr(P, "read_weights"):
        return P.forward(P.read_config(d), P.read_weights(d), tokens).double()
    with open(os.path.join(d, "config.json")) as f:
        cfg = json.load(f)
    f = SafetensorsFile(os.path.join(d, "model.safetensors"))
    return P.forward(cfg, {n: f.read(n) for n in f.names()}, tokens).double()


def agree(entries, logits, prompt, top, off):
    """`off`: how far the engine's logits of a row may lie from `logits` [tokens, V].  A log probability is off by at most twice that; an
    entropy -sum p ln p has the derivative -p_i (ln p_i + H), whose magnitudes add up to at most 2 H <= 2 ln V; 2^-20 stands for the
    32-bit sums over at most a thousand tokens."""
    V = logits.shape[1]
    lp = torch.log_softmax(logits, -1)
    assert len(entries) == len(prompt) - 1
    for i, e in enumerate(entries):
        d = off(logits[i])
        x, t = logits[i], prompt[i + 1]
        eps = 2.0 ** -20 * (1 + float(lp[i].abs().max()))
        assert e["token"] == t and abs(e["logprob"] - float(lp[i, t])) <= 2 * d + eps
        assert abs(e["entropy"] + float((lp[i].exp() * lp[i]).sum())) <= 2 * d * float(torch.log(torch.tensor(float(V)))) + eps
        assert int((x > x[t] + 2 * d).sum()) <= e["rank"] <= int((x >= x[t] - 2 * d).sum()) - (1 if d == 0 else 0)
        assert len(e["top"]) == top
        for j, (token, p) in enumerate(e["top"]):
            assert abs(p - float(lp[i, token])) <= 2 * d + eps
            assert int((x > x[token] + 2 * d).sum()) <= j


@pytest.mark.parametrize("design", DESIGNS)
def test_scores_follow_the_plain_model_whatever_the_portions(model, design):
    d = model(design, "A")
    V = config_from_dict(DESIGNS[design][0]["A"][0]).vocab_size
    g = random.Random(4)
    prompts = [[g.randrange(V) for _ in range(n)] for n in (33, 2, 12)]
    want = [plain(design, d, p) for p in prompts]
    for portion in (1, 5, 64):
        eng = Engine(d, "float32", max_num_seqs=2, max_batched_tokens=portion, max_model_len=48, page_size=8, device="cpu", ops=ref_ops)
        for p, w, entries in zip(prompts, want, eng.score(prompts, top=4)):
            agree(entries, w, p, 4, lambda row: 3e-4)          # (what the designs' own CPU tests hold their logits to)
        assert not eng.runner.processed
        eng.runner.cache.check()
    assert ref_ops.read_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("design", DESIGNS)
def test_scores_on_the_device(model, design, dtype):
    """In 32 bits against the plain model; in both types against 64-bit sums over the logits that `ModelRunner.step` gives for the same portions,
    beside a request that is being served."""
    d = model(design, "C")
    V = config_from_dict(DESIGNS[design][0]["C"][0]).vocab_size
    g = random.Random(4)
    prompts = [[g.randrange(V) for _ in range(n)] for n in (150, 65, 2)]
    eng = Engine(d, dtype, max_num_seqs=3, max_batched_tokens=64, max_model_len=256, page_size=64)
    served = [g.randrange(V) for _ in range(20)]
    alone = eng.generate([served], max_new_tokens=12)[0]
    req = eng.add_request(served, SamplingParams(temperature=0.0, max_new_tokens=12))
    ended = []
    for _ in range(4):
        ended += eng.step()
    scored = eng.score(prompts, top=5)
    r = eng.runner
    for p, entries in zip(prompts, scored):
        r.add_request("again")
        rows = [r.step([("again", p[a:min(a + 64, len(p) - 1)], list(range(min(64, len(p) - 1 - a))))], shape_graphs=False).double().cpu()
                for a in range(0, len(p) - 1, 64)]
        r.end_request("again")
        agree(entries, torch.cat(rows), p, 5, lambda row: 0.0)
        if dtype == "float32":
            agree(entries, plain(design, d, p), p, 5, lambda row: 5e-5 * float(row.abs().max()))    # (as the designs' own tests)
    while eng.has_work():
        ended += eng.step()
    ended += eng.flush()
    got = [x for x in ended if x.request_id == req]
    assert len(got) == 1 and (dtype != "float32" or got[0].output == alone)
    assert not r.processed and r.ops.read_status() == 0
    r.cache.check()
