"""Log probabilities of given tokens, with entropy and the likeliest alternatives, from logits and from hidden states.

``tokens`` cases take rows of logits as a step of the engine leaves them (float32, or bfloat16 as other programs keep them); ``head``
cases take the rows that the output head would be multiplied with, and its weight.  For a row of logits x, NaN counting as minus infinity:

    lse = ln sum exp(x),  logprob = x[token] - lse,  entropy = -sum p ln p  with  p = exp(x - lse),

and the ``top`` largest logits, equal ones by ascending id, minus lse.  A row with nothing above minus infinity has no distribution:
every log probability is minus infinity and the entropy 0.  A token outside the vocabulary (a padded row asks for -1) has minus infinity.

Sizes: the benchmark's vocabulary and widths (151,936; 2,048 and 4,096), its batches of 1, 8 and 64 and its prompt of 2,048 tokens, the
tests' small shapes, and generic ones between.
"""
import math

import torch

own = False
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _tokens(name, rows, vocab, top, held=0, pad=0, dtype="fp32", masked=False):
    """``held``: rows of the buffer that the ``rows`` are picked from (0: all of them, in order); ``pad``: columns between rows."""
    return dict(name=name, op="tokens", rows=rows, vocab=vocab, top=top, held=held, pad=pad, dtype=dtype, masked=masked)


def _head(name, rows, width, vocab, top=0, cap=0.0, dtype="bf16"):
    return dict(name=name, op="head", rows=rows, width=width, vocab=vocab, top=top, cap=cap, dtype=dtype)


def listed():
    return [
        # a single request that decodes with log probabilities: the smallest call
        _tokens("step of 1, top 5", 1, 151936, 5),
        # eight of a step's 64 requests asked for log probabilities, with the twenty likeliest tokens
        _tokens("step, 8 of 64, top 20", 8, 151936, 20, held=64),
        # all requests of a batch of 64
        _tokens("step of 64, top 5", 64, 151936, 5),
        # a prompt of 2,048 tokens whose logits were kept
        _tokens("prompt of 2048", 2048, 151936, 0),
        # many rows of a small model, where a row is a few hundred values
        _tokens("small vocabulary", 1000, 384, 3),
        # constrained decoding: most tokens masked, rows with nothing left, bfloat16 logits at an odd row stride
        _tokens("masked bf16 rows", 333, 50001, 8, pad=6, dtype="bf16", masked=True),
        # the few tokens of an answer scored behind a long prompt (8B's head): one pass over the weights
        _head("answer of 5", 5, 4096, 151936),
        # a short portion on the 1.7B head, with the five likeliest tokens at every place
        _head("portion of 100, top 5", 100, 2048, 151936, top=5),
        # perplexity over the benchmark's prompt on the 8B head
        _head("prompt of 2048, 8b", 2048, 4096, 151936),
        # two prompts at once, one token short, on the 1.7B head: the largest call
        _head("prompts, 4095 rows", 4095, 2048, 151936),
        # a small model with capped logits
        _head("capped, 700 rows", 700, 1024, 20000, cap=30.0),
        # the true 32-bit path, as used to check a model
        _head("fp32, 257 rows, top 1", 257, 1024, 20000, top=1, dtype="fp32"),
    ]


def _between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.5:
        vocab = _between(rng, 257, 160000)
        rows = _between(rng, 1, max(1, min(4096, 2048 * 151936 // vocab)))
        c = _tokens("", rows, vocab, rng.choice((0, 1, 2, 5, 10, 20, 32)), held=rows + rng.randrange(1, 40) if rng.random() < 0.3 else 0,
                    pad=rng.choice((0, 0, 1, 3, 8)), dtype=rng.choice(("fp32", "fp32", "bf16")), masked=rng.random() < 0.3)
    else:
        fp32 = rng.random() < 0.15
        width, vocab = 8 * _between(rng, 8, 128 if fp32 else 640), _between(rng, 257, 32000 if fp32 else 160000)
        rows = _between(rng, 1, max(1, min(512 if fp32 else 8192, 4095 * 2048 * 151936 // (width * vocab))))
        c = _head("", rows, width, vocab, top=rng.choice((0, 0, 1, 5, 8)) if rows <= 256 else 0, cap=30.0 if rng.random() < 0.2 else 0.0,
                  dtype="fp32" if fp32 else "bf16")
    del c["name"]
    return c


LEADERS = 10          # tokens that stand out in every row, as a trained model's do


def _leading(n, vocab, gen):
    """Ids [n, LEADERS] of the tokens that lead a row and what their logits have over the others."""
    ids = torch.randint(0, vocab, (n, LEADERS), generator=gen, device="cuda")
    steps = 0.8 + 0.8 * torch.rand(n, LEADERS, generator=gen, device="cuda")
    return ids, 14 + 10 * torch.rand(n, 1, generator=gen, device="cuda") - steps.cumsum(1)


def _given(ids, vocab, gen, masked=False):
    """The tokens that followed: mostly one of the leading ones, some from anywhere (not where a mask allows few), a few rows that are padding."""
    n = ids.shape[0]
    u = torch.rand(n, generator=gen, device="cuda")
    pick = (6 * torch.rand(n, generator=gen, device="cuda") ** 3).long()
    any_id = torch.randint(0, vocab, (n,), generator=gen, device="cuda")
    t = torch.where((u < 0.8) | masked, ids.gather(1, pick[:, None])[:, 0], any_id)
    return torch.where(u > 0.98, -1, t).to(torch.int32) if n > 1 else t.to(torch.int32)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    n, V, top = case["rows"], case["vocab"], case["top"]
    dtype = DTYPES[case["dtype"]]
    s = dict(case)
    if case["op"] == "tokens":
        held = case["held"] or n
        x = torch.randn(held, V + case["pad"], generator=gen, device="cuda").mul_(1.3)
        ids, lead = _leading(held, V, gen)
        x.scatter_add_(1, ids, lead)
        if case["masked"]:
            keep = torch.rand(held, V + case["pad"], generator=gen, device="cuda") < max(0.02, 96 / V)
            keep.scatter_(1, ids, True)
            low = torch.where(torch.arange(held, device="cuda") % 3 == 0, torch.finfo(dtype).min, -math.inf)
            x = torch.where(keep, x, low[:, None])
            x[5::11] = -math.inf                                   # nothing is allowed here
            x[6::11, : V // 2] = math.nan
        s["logits"] = x.to(dtype)[:, :V]
        s["rows_at"] = torch.randperm(held, generator=gen, device="cuda")[:n].to(torch.int32) if case["held"] else None
        s["tokens"] = _given(ids if s["rows_at"] is None else ids[s["rows_at"].long()], V, gen, case["masked"])
    else:
        H = case["width"]
        w = torch.randn(V, H, generator=gen, device="cuda").mul_(0.02)
        ids, lead = _leading(n, V, gen)
        h = torch.randn(n, H, generator=gen, device="cuda")
        for a in range(0, n, 512):                                 # the leading tokens' directions, by what their logits get
            rows = w[ids[a:a + 512]]
            h[a:a + 512] += torch.einsum("nl,nlh->nh", lead[a:a + 512] / rows.square().sum(-1), rows)
        s["hidden"], s["weight"] = h.to(dtype), w.to(dtype)
        s["tokens"] = _given(ids, V, gen)
    if own:
        _buffers(s)
    return s


def _buffers(s):
    """What a program keeps for the calls: the results' places, the error word, the scratch."""
    from airun_b200.engine.batch import Workspace
    n, top = s["rows"], s["top"]
    s["logprob"], s["entropy"] = (torch.empty(n, device="cuda") for _ in range(2))
    s["top_ids"] = torch.empty(n, top, dtype=torch.int32, device="cuda") if top else None
    s["top_logprobs"] = torch.empty(n, top, device="cuda") if top else None
    s["err"] = torch.zeros(1, dtype=torch.int32, device="cuda")
    s["ws"] = Workspace(torch.device("cuda"))


def _plain(x, tokens, top):
    """Everything from logits x [n, V] in 32 bits."""
    V = x.shape[1]
    x = torch.where(torch.isnan(x), -math.inf, x) + 0.0
    m = x.amax(1, keepdim=True)
    some = m > -math.inf
    d = torch.where(x > -math.inf, x - torch.where(some, m, 0.0), -math.inf)
    e = torch.exp(d)
    total = e.sum(1, keepdim=True)
    lse = torch.where(some, m + torch.log(total), 0.0)
    u = torch.where(e > 0, e * d, 0.0).sum(1)
    t = tokens.long()
    got = x.gather(1, t.clamp(0, V - 1)[:, None]) - lse
    out = {"logprob": torch.where((t >= 0) & (t < V), got[:, 0], -math.inf),
           "entropy": torch.where(some[:, 0], torch.log(total[:, 0]) - u / total[:, 0], 0.0)}
    if top:
        bits = x.view(torch.int32)
        key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long() * (1 << 32) + ((1 << 32) - 1 - torch.arange(V, device=x.device))
        ids = 0xFFFFFFFF - (torch.topk(key, top, dim=1).values & 0xFFFFFFFF)
        out["top_ids"], out["top_logprobs"] = ids.to(torch.int32), x.gather(1, ids) - lse
    return out


def run(state):
    s = state
    if own:
        from airun_b200.kernels import ops
        if s["op"] == "tokens":
            ops.token_logprobs(s["logits"], s["tokens"], s["logprob"], entropy=s["entropy"], top_ids=s["top_ids"],
                               top_logprobs=s["top_logprobs"], rows=s["rows_at"], err=s["err"])
        else:
            s["ws"].reset()
            ops.head_logprobs(s["hidden"], s["weight"], s["tokens"], s["logprob"], s["err"], entropy=s["entropy"], top_ids=s["top_ids"],
                              top_logprobs=s["top_logprobs"], soft_cap=s["cap"] or None, ws=s["ws"])
        out = {"logprob": s["logprob"], "entropy": s["entropy"]}
        return dict(out, top_ids=s["top_ids"], top_logprobs=s["top_logprobs"]) if s["top"] else out
    if s["op"] == "tokens":
        x = s["logits"] if s["rows_at"] is None else s["logits"][s["rows_at"].long()]
        return _plain(x.float(), s["tokens"], s["top"])
    x = s["hidden"].float() @ s["weight"].float().t()
    if s["cap"]:
        x = s["cap"] * torch.tanh(x / s["cap"])
    return _plain(x, s["tokens"], s["top"])


def work(case):
    n, V, e = case["rows"], case["vocab"], 4 if case["dtype"] == "fp32" else 2
    out = n * (4 + 8 + 8 * case["top"])
    if case["op"] == "tokens":
        return {"bytes": n * V * e + out, "flops": 4 * n * V}
    return {"bytes": (n + V) * case["width"] * e + out, "flops": 2 * n * V * case["width"]}


def exact(case, seed):
    s = prepare(case, seed)
    n, V, top = case["rows"], case["vocab"], case["top"]
    parts = []
    step = max(1, (1 << 28) // V)                                  # rows whose logits in 64 bits are 2 GiB
    for a in range(0, n, step):
        t = s["tokens"][a:a + step].long()
        if case["op"] == "tokens":
            at = torch.arange(a, min(n, a + step), device="cuda") if s["rows_at"] is None else s["rows_at"][a:a + step].long()
            z = s["logits"][at].double().nan_to_num(nan=-math.inf, posinf=math.inf, neginf=-math.inf)
        else:
            z = torch.mm(s["hidden"][a:a + step].double(), s["weight"].double().t())
            if case["cap"]:
                z = torch.tanh(z / case["cap"]) * case["cap"]
        lp = z - torch.logsumexp(z, 1, keepdim=True)               # a row of minus infinities gives NaN here
        lp = lp.nan_to_num(nan=-math.inf, neginf=-math.inf)
        p = lp.exp()
        logprob = torch.full((t.shape[0],), -math.inf, dtype=torch.float64, device="cuda")
        real = ((t >= 0) & (t < V)).nonzero()[:, 0]
        logprob[real] = lp[real, t[real]]
        parts.append((logprob, -torch.special.xlogy(p, p).sum(1), lp.sort(1, descending=True).values[:, :top] if top else None))
    out = {"logprob": torch.cat([p[0] for p in parts]), "entropy": torch.cat([p[1] for p in parts])}
    if top:
        out["top_ids"], out["top_logprobs"] = None, torch.cat([p[2] for p in parts])
    return out
