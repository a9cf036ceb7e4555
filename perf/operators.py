"""Three operators of a drafted decode step, as cases that can be timed: what a draft model's small products, the target's
attention over a prompt that the whole batch begins with, and the test of the drafted tokens cost.

``int4``     rows of bfloat16 times a matrix kept in 4 bits with a scale (and a zero point) per group of its columns
``prefix``   attention of new tokens whose sequences share their first pages in the cache: those pages are read once for all
``verify``   drafted tokens held to the target's distribution with given random numbers, and the token that follows them

A case says the sizes, the seed everything else.  Where ``own`` is false ``run`` computes the operator from elementary torch
operations; where it is true it makes the calls of ``rust_inference_amd.kernels.ops``.
"""
import math
import random

import torch

own = False

PAGE = 32                        # tokens of a page of the cache


def _int4(name, rows, n, k, group, zeros, scale_type, out_type):
    return {"name": name, "op": "int4", "rows": rows, "n": n, "k": k, "group": group, "zeros": zeros, "scale_type": scale_type,
            "out_type": out_type}


def _prefix(name, seqs, new, heads, kv_heads, dim, shared, low, high):
    return {"name": name, "op": "prefix", "seqs": seqs, "new": new, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "shared": shared, "low": low, "high": high}


def _verify(name, seqs, low, high, vocab, temperature, draft):
    return {"name": name, "op": "verify", "seqs": seqs, "low": low, "high": high, "vocab": vocab, "temperature": temperature,
            "draft": draft}


def listed():
    return [
        # one token of one user through an attention output matrix: a few microseconds of weights, latency counts
        _int4("one_row_4096", 1, 4096, 4096, 128, False, "bfloat16", "bfloat16"),
        # the gate and up rows of a feed-forward for a few users, with zero points
        _int4("gate_up_8_rows", 8, 24576, 4096, 128, True, "bfloat16", "bfloat16"),
        # the logits of a batch: the largest matrix of a model, float32 out
        _int4("logits_16_rows", 16, 151936, 4096, 64, True, "float32", "float32"),
        # rows of a drafted step through a matrix of odd sizes, small groups of which the last is short
        _int4("odd_45_rows", 45, 5001, 2568, 32, True, "bfloat16", "bfloat16"),
        # a few users of a small model behind a system prompt
        _prefix("four_users", 4, 1, 16, 8, 128, 1024, 1, 200),
        # a full batch behind a long system prompt, every sequence with an answer of its own
        _prefix("batch_64", 64, 1, 32, 8, 128, 8192, 64, 1500),
        # the same prompt with drafts: up to five new tokens a sequence
        _prefix("drafted_16", 16, 5, 32, 8, 128, 4096, 20, 900),
        # many questions about one long document, eight query heads a key head
        _prefix("document_131072", 32, 1, 64, 8, 128, 131072, 30, 600),
        # one user's four drafts, with the draft model's logits
        _verify("one_user", 1, 4, 4, 151936, 0.8, True),
        # a full batch of four drafts each
        _verify("batch_64_drafts", 64, 4, 4, 151936, 1.0, True),
        # drafts looked up in the prompt, none to eight of them: no distribution of their own, a vocabulary of odd size
        _verify("looked_up", 16, 0, 8, 50021, 0.7, False),
        # greedy decoding: a draft stands while it is the target's best token
        _verify("greedy_32", 32, 5, 5, 151936, 0.0, False),
    ]


def _spread(rng, low, high):
    """A whole number from ``low`` to ``high``, spread over the logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(("int4", "prefix", "verify"))
    if op == "int4":
        k = 8 * _spread(rng, 32, 1600)
        n = min(_spread(rng, 200, 60000), 200_000_000 // k)
        case = _int4("", _spread(rng, 1, 64), n, k, rng.choice((32, 64, 128, 128, 256)), rng.random() < 0.6,
                     rng.choice(("bfloat16", "float32")), rng.choice(("bfloat16", "bfloat16", "float32")))
    elif op == "prefix":
        kv_heads = rng.choice((1, 2, 4, 8))
        heads, new = kv_heads * rng.choice((1, 2, 3, 4, 5, 8)), rng.choice((1, 1, 2, 4, 7))
        seqs = _spread(rng, 1, 64 // new)
        low = _spread(rng, new, 400)
        case = _prefix("", seqs, new, heads, kv_heads, rng.choice((64, 128, 128)), PAGE * _spread(rng, 1, 1024), low,
                       low + rng.randint(0, 1200))
    else:
        low = rng.choice((0, 1, 2, 4))
        case = _verify("", _spread(rng, 1, 36), low, low + rng.randint(0, 3), _spread(rng, 1000, 151936),
                       rng.choice((0.0, 0.5, 0.8, 1.0, 1.3)), rng.random() < 0.6)
    del case["name"]
    return case


# ---------------------------------------------------------------- inputs
def _counts(case):
    """Drafts of every sequence."""
    r = random.Random(repr((case["seqs"], case["low"], case["high"])))
    return [r.randint(case["low"], case["high"]) for _ in range(case["seqs"])]


def _lengths(case):
    """(new tokens, tokens behind the shared ones with the new ones) of every sequence."""
    r = random.Random(repr((case["seqs"], case["low"], case["high"], case["new"])))
    out = []
    for i in range(case["seqs"]):
        new = case["new"] if i == 0 else r.randint(1, case["new"])
        out.append((new, max(new, r.randint(case["low"], case["high"]))))
    return out


def _starts(counts, device):
    cu = [0]
    for n in counts:
        cu.append(cu[-1] + n)
    return torch.tensor(cu, dtype=torch.int32, device=device)


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def prepare(case, seed):
    """The inputs a user's program holds before the call: the weights as a checkpoint stores them, the cache with the new tokens'
    keys and values in it, or the logits of a step."""
    g = torch.Generator("cuda").manual_seed(seed)
    s = dict(case)
    if case["op"] == "int4":
        rows, n, k, group = case["rows"], case["n"], case["k"], case["group"]
        s["x"] = _normal(g, rows, k).to(torch.bfloat16)
        s["codes"] = torch.randint(0, 256, (n, k // 2), generator=g, device="cuda", dtype=torch.uint8)
        groups = -(-k // group)
        s["scales"] = (0.004 + 0.008 * torch.rand(n, groups, generator=g, device="cuda")).to(getattr(torch, case["scale_type"]))
        s["zero_points"] = torch.randint(5, 11, (n, groups), generator=g, device="cuda", dtype=torch.uint8) if case["zeros"] else None
        return s
    if case["op"] == "prefix":
        lens, heads, kv, dim, shared = _lengths(case), case["heads"], case["kv_heads"], case["dim"], case["shared"]
        first = shared // PAGE
        own_pages = [-(-m // PAGE) for _, m in lens]
        pages, width = first + sum(own_pages), first + max(own_pages)
        order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32).cpu()
        table, at = torch.zeros((len(lens), width), dtype=torch.int32), first
        for b, m in enumerate(own_pages):
            table[b, :first] = order[:first]
            table[b, first:first + m] = order[at:at + m]
            at += m
        s["k_pages"] = _normal(g, pages, kv, PAGE, dim).to(torch.bfloat16)
        s["v_pages"] = _normal(g, pages, kv, dim, PAGE).to(torch.bfloat16)
        counts = [n for n, _ in lens]
        s["qkv"] = (1.5 * _normal(g, sum(counts), (heads + 2 * kv) * dim)).to(torch.bfloat16)
        s["page_table"], s["cu_seqlens"] = table.cuda(), _starts(counts, "cuda")
        s["tok_pos"] = torch.tensor([shared + m - n + i for n, m in lens for i in range(n)], dtype=torch.int32, device="cuda")
        s["max_len"], s["max_new"], s["scale"] = shared + max(m for _, m in lens), max(counts), dim ** -0.5
        return s
    counts, vocab, temperature = _counts(case), case["vocab"], case["temperature"]
    rows = sum(counts) + len(counts)
    s["cu_seqlens"] = _starts([n + 1 for n in counts], "cuda")
    s["logits"] = 2.5 * _normal(g, rows, vocab)
    near = s["logits"] + 0.8 * _normal(g, rows, vocab)            # what another, smaller model says of the same place
    noise = -torch.log(-torch.log(torch.rand(rows, vocab, generator=g, device="cuda").clamp_(1e-7, 1 - 1e-7)))
    drawn = (near / temperature + noise if temperature > 0 else near).argmax(1)      # (a draw from the draft's distribution)
    s["tokens"] = drawn.roll(1).to(torch.int32)                    # token j was drawn from the row before it
    s["draft_logits"] = near.roll(1, 0).contiguous() if case["draft"] else None      # row j: what token j was drawn from
    s["uniform"] = torch.rand(rows, generator=g, device="cuda") if temperature > 0 else None
    return s


# ---------------------------------------------------------------- the passes
def run(s):
    if s["op"] == "int4":
        return _run_int4(s)
    if s["op"] == "prefix":
        return _run_prefix(s)
    return _run_verify(s)


def _run_int4(s):
    out_type = getattr(torch, s["out_type"])
    if own:
        from rust_inference_amd.kernels import ops
        return ops.gemm_int4_bf16(s["x"], s["codes"], s["scales"], s["group"], s["zero_points"], out_type)
    codes, group = s["codes"], s["group"]
    n, k = codes.shape[0], 2 * codes.shape[1]
    q = torch.stack((codes & 15, codes >> 4), 2).view(n, k).float()
    scales = s["scales"].float().repeat_interleave(group, 1)[:, :k]
    zeros = 8.0 if s["zero_points"] is None else s["zero_points"].float().repeat_interleave(group, 1)[:, :k]
    return torch.matmul(s["x"].float(), q.sub_(zeros).mul_(scales).t()).to(out_type)


def _run_prefix(s):
    heads, kv, dim, shared, seqs = s["heads"], s["kv_heads"], s["dim"], s["shared"], s["seqs"]
    if own:
        from rust_inference_amd.kernels import ops
        return ops.attention_shared_bf16(s["qkv"], s["k_pages"], s["v_pages"], s["cu_seqlens"], s["tok_pos"], s["page_table"], seqs,
                                         s["max_new"], shared, s["max_len"], heads, kv, dim, s["scale"])
    tokens, per, first = s["qkv"].shape[0], heads // kv, shared // PAGE
    q = (s["qkv"][:, :heads * dim].float() * s["scale"]).view(tokens, kv, per, dim).transpose(0, 1).contiguous()
    table = s["page_table"].long()
    # the shared keys, once for all tokens
    k = s["k_pages"][table[0, :first]].float().transpose(0, 1).reshape(kv, shared, dim)
    v = s["v_pages"][table[0, :first]].float().permute(1, 0, 3, 2).reshape(kv, shared, dim)
    far = torch.matmul(q.view(kv, tokens * per, dim), k.transpose(1, 2).contiguous()).view(kv, tokens, per, shared)
    # every token's own ones
    reach = (table.shape[1] - first) * PAGE
    seq = torch.bucketize(torch.arange(tokens, device=table.device), s["cu_seqlens"][1:].long(), right=True)
    ok = s["k_pages"][table[:, first:]].float().permute(2, 0, 1, 3, 4).reshape(kv, seqs, reach, dim)[:, seq]
    ov = s["v_pages"][table[:, first:]].float().permute(2, 0, 1, 4, 3).reshape(kv, seqs, reach, dim)[:, seq]
    near = torch.matmul(q, ok.transpose(2, 3).contiguous())
    ahead = shared + torch.arange(reach, device=table.device)[None, :] > s["tok_pos"].long()[:, None]
    near = near.masked_fill(ahead[None, :, None, :], -math.inf)
    top = torch.maximum(far.amax(3, keepdim=True), near.amax(3, keepdim=True))
    far, near = far.sub_(top).exp_(), near.sub_(top).exp_()
    total = far.sum(3, keepdim=True) + near.sum(3, keepdim=True)
    out = torch.matmul(far.view(kv, tokens * per, shared), v).view(kv, tokens, per, dim) + torch.matmul(near, ov)
    return (out / total).transpose(0, 1).reshape(tokens, heads * dim).to(torch.bfloat16)


def _probabilities(logits, temperature):
    x = logits.double().div_(temperature)
    e = x.sub_(x.amax(1, keepdim=True)).exp_()
    return e.div_(e.sum(1, keepdim=True))


def _run_verify(s):
    logits, draft, tokens, cu, temperature = s["logits"], s["draft_logits"], s["tokens"], s["cu_seqlens"], s["temperature"]
    if own:
        from rust_inference_amd.kernels import ops
        return ops.verify_drafts(logits, tokens, cu, s["uniform"], temperature, draft)
    cu = cu.long()
    first, last, rows = cu[:-1], cu[1:] - 1, logits.shape[0]
    row = torch.arange(rows, device=cu.device)
    seq = torch.bucketize(row, cu[1:], right=True)
    drafted = tokens.long().roll(-1)                               # the draft that a row's distribution is asked about
    if temperature <= 0:
        best = logits.argmax(1)
        stands = best == drafted
    else:                                                          # in 64 bits: a draw next to a border must fall on its own side
        p = _probabilities(logits, temperature)
        at = p.gather(1, drafted[:, None])[:, 0]
        said = _probabilities(draft, temperature).roll(-1, 0) if draft is not None else None
        of = said.gather(1, drafted[:, None])[:, 0] if draft is not None else torch.ones_like(at)
        stands = s["uniform"].double() * of < at
    fails = torch.where(stands & (row < last[seq]), rows, row)     # a sequence's last row has no draft to stand
    stop = torch.full_like(first, rows).scatter_reduce(0, seq, fails, "amin")
    accepted = stop - first
    if temperature <= 0:
        token = best[stop]
    else:
        left = p[stop]
        rejected = (stop < last)[:, None]
        if draft is not None:
            less = (left - said[stop]).clamp_(min=0)
        else:
            less = left.scatter(1, drafted[stop][:, None], 0.0)
        left = torch.where(rejected & (less.sum(1, keepdim=True) > 0), less, left)
        upto = left.cumsum(1)
        token = (upto <= s["uniform"].double()[last, None] * left.sum(1, keepdim=True)).sum(1)
        some = left > 0
        token = torch.minimum(token, logits.shape[1] - 1 - some.flip(1).to(torch.uint8).argmax(1))
    out = torch.where(row < stop[seq], drafted, torch.where(row == stop[seq], token[seq], -1))
    return accepted.to(torch.int32), out.to(torch.int32)


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    if case["op"] == "int4":
        rows, n, k, groups = case["rows"], case["n"], case["k"], -(-case["k"] // case["group"])
        size = {"bfloat16": 2, "float32": 4}
        return {"bytes": n * k // 2 + n * groups * (size[case["scale_type"]] + (1 if case["zeros"] else 0)) + 2 * rows * k
                + rows * n * size[case["out_type"]], "flops": 2 * rows * n * k}
    if case["op"] == "prefix":
        lens, heads, kv, dim, shared = _lengths(case), case["heads"], case["kv_heads"], case["dim"], case["shared"]
        tokens, own_keys = sum(n for n, _ in lens), sum(m for _, m in lens)
        seen = sum(shared + m - n + i + 1 for n, m in lens for i in range(n))
        return {"bytes": 4 * kv * dim * (shared + own_keys) + 4 * tokens * heads * dim, "flops": 4 * heads * dim * seen}
    counts = _counts(case)
    rows = sum(counts) + len(counts)
    read = rows + (sum(counts) if case["draft"] and case["temperature"] > 0 else 0)
    return {"bytes": 4 * read * case["vocab"] + 12 * rows + 8 * len(counts), "flops": 4 * read * case["vocab"]}


# ---------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "int4":
        # out[m, n] = sum over the groups g of scale[n, g] (sum over k in g of x[m, k] code[n, k] - zero[n, g] sum over k in g of x[m, k])
        x, group = s["x"].double(), case["group"]
        out = torch.zeros(case["rows"], case["n"], dtype=torch.float64, device="cuda")
        for at in range(0, case["k"], group):
            part = s["codes"][:, at // 2:(at + group) // 2]
            xs, i = x[:, at:at + group], at // group
            sums = xs[:, 0::2] @ (part & 15).double().t() + xs[:, 1::2] @ (part >> 4).double().t()
            zero = s["zero_points"][:, i].double() if case["zeros"] else torch.full((case["n"],), 8.0, dtype=torch.float64, device="cuda")
            out += s["scales"][:, i].double() * (sums - xs.sum(1, keepdim=True) * zero)
        return out
    if case["op"] == "prefix":
        # a sequence after the other, key head by key head, over all its keys as one row of them
        lens, heads, kv, dim, shared = _lengths(case), case["heads"], case["kv_heads"], case["dim"], case["shared"]
        out, at = [], 0
        for b, (new, own_len) in enumerate(lens):
            length = shared + own_len
            pages = s["page_table"][b, :-(-length // PAGE)].long()
            rows = []
            for h in range(kv):
                keys = s["k_pages"][pages, h].reshape(-1, dim)[:length].double()
                values = s["v_pages"][pages, h].transpose(1, 2).reshape(-1, dim)[:length].double()
                cols = slice(h * (heads // kv) * dim, (h + 1) * (heads // kv) * dim)
                q = s["qkv"][at:at + new, cols].double().view(-1, dim)
                score = (q @ keys.t()).view(new, heads // kv, length) / math.sqrt(dim)
                for i in range(new):
                    score[i, :, length - new + i + 1:] = -math.inf
                weight = torch.exp(score - torch.logsumexp(score, 2, keepdim=True))
                rows.append((weight.view(-1, length) @ values).view(new, -1))
            out.append(torch.cat(rows, 1))
            at += new
        return torch.cat(out, 0)
    return None                                                    # (its outputs are whole numbers)
