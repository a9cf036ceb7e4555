"""Drafted steps through the engine: a step whose tokens are a sequence's last one and its drafts, all rows wanted, verified on the
device, the cache advanced by what stands."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def greedy(engine, prompts, count):
    """The best token after each prompt and after every token since, one a step."""
    slots = [engine.cache.acquire() for _ in prompts]
    fed, out = [list(p) for p in prompts], [[] for _ in prompts]
    for _ in range(count):
        logits = engine.step(list(zip(slots, fed, ["last"] * len(slots))))
        fed = [[int(t)] for t in logits.argmax(1).tolist()]
        for kept, new in zip(out, fed):
            kept += new
    for s in slots:
        engine.cache.release(s)
    return out


@pytest.mark.parametrize("name", ["A", "B", "C"])
@pytest.mark.parametrize("temperature", [0.0, 0.8])
def test_drafted_steps_go_on_as_single_ones_do(model_dirs, name, temperature):
    """Drafts are the tokens that greedy steps gave, some of them changed, of different numbers a sequence, none for some.  With
    temperature 0 every sequence is the one of greedy steps, whatever fell.  Above it numbers of 0 let every draft stand that
    has any weight."""
    from rust_inference_amd.engine.replay import engine_for_trace
    from rust_inference_amd.engine.step import StepEntry
    from rust_inference_amd.kernels import ops
    from rust_inference_amd.parts import load_model
    model = load_model(model_dirs[name], torch.float32)
    vocab, rng = model.spec.vocab_size, np.random.default_rng(7)
    engine = engine_for_trace(model, 1024)
    cache, count = engine.cache, 24
    prompts = [[int(t) for t in rng.integers(0, vocab, n)] for n in (5, 31, 33, 1)]
    best = greedy(engine, prompts, count + 8)
    slots = [cache.acquire() for _ in prompts]
    engine.step([(s, p[:-1], "none") for s, p in zip(slots, prompts) if len(p) > 1])
    got, last = [[] for _ in prompts], [p[-1] for p in prompts]
    fell = 0
    while min(map(len, got)) < count:
        live = [b for b in range(len(prompts)) if len(got[b]) < count]
        drafts = []
        for b in live:
            d = best[b][len(got[b]):len(got[b]) + int(rng.integers(0, 6))]
            if d and rng.random() < 0.4:
                at = int(rng.integers(0, len(d)))
                d[at] = (d[at] + 1) % vocab
            drafts.append(d)
        entries = [StepEntry(slots[b], [last[b]] + d, "all") for b, d in zip(live, drafts)]
        ctx = engine.build_context(entries)
        logits = model.forward(ctx, cache)
        uniform = torch.zeros(ctx.T, device=logits.device) if temperature > 0 else None
        accepted, out = ops.verify_drafts(logits, ctx.tokens, ctx.cu_seqlens, uniform, temperature)
        accepted, out = accepted.tolist(), out.tolist()
        cache.commit(ctx.slot_list, [n + 1 for n in accepted])
        at = 0
        for b, d, n in zip(live, drafts, accepted):
            rows = out[at:at + len(d) + 1]
            assert rows[:n] == d[:n] and rows[n] >= 0 and rows[n + 1:] == [-1] * (len(d) - n)
            if temperature > 0:
                assert n == len(d)
            got[b] += rows[:n + 1]
            last[b] = rows[n]
            fell += len(d) - n
            assert cache.length(slots[b]) == len(prompts[b]) - 1 + len(got[b])
            at += len(d) + 1
        if temperature > 0:                                   # (the text goes on as another one)
            break
        cache.check_consistent()
    if temperature == 0:
        assert fell > 0
        for b in range(len(prompts)):
            assert got[b] == best[b][:len(got[b])]
    for s in slots:
        cache.release(s)
    cache.check_consistent()
