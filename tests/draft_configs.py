"""Two tiny models whose mixers are attention alone, so that trees of drafted tokens run through them: LFM2 layers of full attention."""

TREES_A = {
    "architectures": ["Lfm2ForCausalLM"], "hidden_size": 64, "num_hidden_layers": 3, "layer_types": ["full_attention"] * 3,
    "num_attention_heads": 4, "num_key_value_heads": 2, "head_dim": 16, "block_ff_dim": 192, "block_auto_adjust_ff_dim": False,
    "vocab_size": 61, "rope_theta": 10000.0, "conv_L_cache": 3, "conv_bias": False, "use_qk_norm": True, "norm_eps": 1e-5,
    "tie_embedding": True, "max_position_embeddings": 128,
}

# head size 64: the tensor-core kernels in bfloat16
TREES_B = {**TREES_A, "hidden_size": 256, "num_attention_heads": 4, "num_key_value_heads": 2, "head_dim": 64, "block_ff_dim": 512, "vocab_size": 199,
           "max_position_embeddings": 2048}


def draft(g, truth, n, vocab):
    """A tree of n tokens behind truth[0]: some of the true continuation, wrong branches beside it, now and then a twin."""
    tokens, parents, on_path, depth = [truth[0]], [-1], 0, 0
    while len(tokens) < n:
        if depth + 1 < len(truth) and g.random() < 0.4:
            tokens.append(truth[depth + 1])
            parents.append(on_path)
            on_path, depth = len(tokens) - 1, depth + 1
        elif len(tokens) > 1 and g.random() < 0.2:
            tokens.append(tokens[-1])
            parents.append(parents[-1])
        else:
            tokens.append(g.randrange(vocab))
            parents.append(g.randrange(len(tokens) - 1))
    return tokens, parents


def speculate(runner, prompts, new, truths, g, vocab, most=9):
    """Generate `new` greedy tokens for every prompt by checking drafted trees, several requests a step."""
    out, pending = {}, {}
    for rid, p in prompts.items():
        runner.add_request(rid)
        runner.step([(rid, p[:-1], [])]) if len(p) > 1 else None
        out[rid], pending[rid] = [], p[-1]
    steps = 0
    while pending:
        entries = []
        for rid in sorted(pending):
            truth = [pending[rid]] + truths[rid][len(out[rid]):]
            entries.append((rid, *draft(g, truth, g.randint(1, most), vocab)))
        for (rid, _, _), toks in zip(entries, runner.verify(entries)):
            assert toks
            out[rid] += toks
            pending[rid] = toks[-1]
        steps += 1
        for rid in [r for r in pending if len(out[r]) >= new]:
            del pending[rid]
            runner.end_request(rid)
    runner.cache.check()
    return {r: t[:new] for r, t in out.items()}, steps
