"""The operators of a step that checks a tree of drafted tokens, as measurable cases.

A request offers its last token and a tree of guesses behind it (drafted by a smaller model or copied from the prompt) in
one step.  The step's attention lets a token see what is cached before the step and, of the step's own tokens, the ones its
mask names (its ancestors): ``tree_attention``.  Its logits become the distributions that sampling draws from:
``probabilities``.  The guesses are accepted or rejected so that every token is distributed as if it had been drawn one at
a time: ``verify_drafts``.  What the accepted path stored moves together behind the cached tokens: ``keep_tokens``.

With ``own`` false ``run`` works the operators out in elementary torch operations, with it true through the package.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEVICE = "cuda:0"
PAGE = 16               # tokens to a page of the cache, the engine's default
DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


# --------------------------------------------------------------------------------------------------------- the cases
def _attention(name, requests, nodes, context, heads, kv_heads, dim, dtype="bfloat16"):
    """``nodes``: tokens of the largest tree, ``context``: keys of the longest request; the others are smaller."""
    c = {"kind": "tree_attention", "requests": requests, "nodes": nodes, "context": context, "heads": heads,
         "kv_heads": kv_heads, "dim": dim, "dtype": dtype}
    return dict(c, name=name) if name else c


def _probabilities(name, rows, vocab, temperature, top_k, top_p):
    c = {"kind": "probabilities", "rows": rows, "vocab": vocab, "temperature": temperature, "top_k": top_k, "top_p": top_p}
    return dict(c, name=name) if name else c


def _verify(name, requests, nodes, width, vocab, drawn):
    """``width``: guesses behind one token at most; ``drawn``: the guesses come with the distribution they were drawn from."""
    c = {"kind": "verify_drafts", "requests": requests, "nodes": nodes, "width": width, "vocab": vocab, "drawn": drawn}
    return dict(c, name=name) if name else c


def _keep(name, requests, layers, kv_heads, dim, context, nodes, depth, dtype="bfloat16"):
    c = {"kind": "keep_tokens", "requests": requests, "layers": layers, "kv_heads": kv_heads, "dim": dim, "context": context,
         "nodes": nodes, "depth": depth, "dtype": dtype}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one user of the small model, a short conversation, a small tree: nothing but latency
        _attention("attention_one", 1, 8, 200, 14, 2, 64),
        # an ordinary batch at the 7B sizes: trees of up to 16 behind up to two thousand tokens
        _attention("attention_batch", 8, 16, 2000, 28, 4, 128),
        # a few long documents at the 32B sizes with large trees: as many products as keys to read
        _attention("attention_long", 4, 63, 16011, 40, 8, 128),
        # the 32-bit path
        _attention("attention_float", 6, 13, 700, 14, 2, 64, "float32"),
        # the rows of one user's small tree, sampled as the engine's examples sample: temperature, top-k and top-p
        _probabilities("probabilities_one", 8, 151936, 0.8, 50, 0.9),
        # the rows of a batch of trees, top-p alone
        _probabilities("probabilities_batch", 130, 152064, 0.8, 0, 0.9),
        # temperature alone, an odd vocabulary
        _probabilities("probabilities_plain", 33, 100003, 1.0, 0, 1.0),
        # one user's small tree, two guesses a token
        _verify("verify_one", 1, 8, 2, 151936, True),
        # a batch of large trees, up to four guesses a token
        _verify("verify_batch", 16, 31, 4, 152064, True),
        # guesses copied from the prompt: chains without a distribution
        _verify("verify_chain", 8, 6, 1, 151936, False),
        # what one user's accepted guesses stored, all layers of the small model
        _keep("keep_one", 1, 24, 2, 64, 333, 16, 5),
        # a full batch at the 32B sizes
        _keep("keep_batch", 32, 64, 8, 128, 96, 32, 8),
    ]


def _spread(rng, low, high):
    """A whole number from low to high, as likely in every part of the range's logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 0.5))))))


def draw(rng):
    kind = rng.choice(["tree_attention", "probabilities", "verify_drafts", "keep_tokens"])
    if kind == "tree_attention":
        heads, kv_heads, dim = rng.choice([(14, 2, 64), (7, 1, 64), (28, 4, 128), (40, 8, 128), (6, 2, 32), (4, 4, 128)])
        dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
        nodes = _spread(rng, 1, 63)
        requests = _spread(rng, 1, 32)
        most = 4 * 63 * 16011 * 40 * 128 // (heads * dim * nodes * requests) // (1 if dtype == "bfloat16" else 16)
        context = _spread(rng, nodes, max(nodes, min(16011, most, 131072 // requests)))
        return _attention(None, requests, nodes, context, heads, kv_heads, dim, dtype)
    if kind == "probabilities":
        top_k, top_p = rng.choice([(50, 0.9), (0, 0.9), (0, 1.0), (20, 1.0), (200, 0.95)])
        vocab = _spread(rng, 1000, 152064)
        rows = _spread(rng, 1, 130)
        return _probabilities(None, rows, vocab, rng.choice([0.7, 0.8, 1.0]), top_k, top_p)
    if kind == "verify_drafts":
        vocab = _spread(rng, 1000, 152064)
        return _verify(None, _spread(rng, 1, 16), _spread(rng, 2, 31), rng.choice([1, 2, 3, 4]), vocab, rng.random() < 0.7)
    layers, kv_heads, dim = rng.choice([(24, 2, 64), (28, 4, 128), (64, 8, 128), (3, 2, 32)])
    dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
    depth = _spread(rng, 1, 8)
    nodes = rng.randint(2 * depth + 1, 32)
    most = 96 if dtype == "bfloat16" else 48
    return _keep(None, _spread(rng, 1, 32), layers, kv_heads, dim, rng.randint(nodes, most), nodes, depth, dtype)


def _lengths(case):
    """Tokens of every request's tree and keys it holds with them: the first request has the most of both, the others fewer.
    They belong to the case and not to the seed."""
    rng = random.Random(f"{case['requests']} {case['nodes']} {case['context']}")
    trees, contexts = [case["nodes"]], [case["context"]]
    for _ in range(case["requests"] - 1):
        trees.append(rng.randint((case["nodes"] + 1) // 2, case["nodes"]))
        contexts.append(rng.randint(max(trees[-1], case["context"] // 2), case["context"]))
    return trees, contexts


def work(case):
    """What an operator cannot do without: every input it needs read once, its results written once."""
    if case["kind"] == "tree_attention":
        size = 2 if case["dtype"] == "bfloat16" else 4
        trees, contexts = _lengths(case)
        tokens = sum(trees)
        keys = sum(contexts) * case["kv_heads"] * case["dim"] * 2 * size
        return {"bytes": keys + 2 * tokens * case["heads"] * case["dim"] * size + tokens * 4 * ((case["nodes"] + 31) // 32),
                "flops": 4 * case["dim"] * case["heads"] * sum(n * c for n, c in zip(trees, contexts))}
    if case["kind"] == "probabilities":
        values = case["rows"] * case["vocab"]
        return {"bytes": 8 * values, "flops": 4 * values}
    if case["kind"] == "verify_drafts":     # the row a request's token is drawn from, of the target and of the draft
        values = case["requests"] * case["vocab"] * (2 if case["drawn"] else 1)
        return {"bytes": 4 * values, "flops": 3 * values}
    size = 2 if case["dtype"] == "bfloat16" else 4
    # half of the depth is accepted on average, and the first of the path stays where it is
    moved = case["requests"] * (case["depth"] + 1) // 2
    return {"bytes": 2 * moved * case["layers"] * 2 * case["kv_heads"] * case["dim"] * size, "flops": 0}


# --------------------------------------------------------------------------------------------------------- the inputs
def _tree(rng, nodes, width):
    """Parents of a tree's tokens in the order of their numbers, which is breadth first; the first is the root (-1)."""
    parents, open_, at = [-1], [0], 0
    while len(parents) < nodes:
        for _ in range(rng.randint(1, width)):
            if len(parents) < nodes:
                parents.append(open_[at])
                open_.append(len(parents) - 1)
        at += 1
    return parents


def _masks(parents, words):
    """A row of bits for every token: itself and its ancestors."""
    rows = []
    for n, p in enumerate(parents):
        rows.append((rows[p] if p >= 0 else 0) | (1 << n))
    out = []
    for bits in rows:
        for w in range(words):
            word = (bits >> (32 * w)) & 0xFFFFFFFF
            out.append(word - (1 << 32) if word >= 1 << 31 else word)
    return out


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _starts(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return out


def _tables(g, contexts):
    """Pages dealt out at random, as a cache in use has them; page 0 belongs to nobody."""
    pages = [-(-c // PAGE) for c in contexts]
    order = torch.randperm(sum(pages), generator=g, device=DEVICE).int() + 1
    table = torch.zeros((len(contexts), max(pages)), dtype=torch.int32, device=DEVICE)
    at = 0
    for r, n in enumerate(pages):
        table[r, :n] = order[at:at + n]
        at += n
    return table, sum(pages) + 1


def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    rng = random.Random(seed)
    return {"tree_attention": _prepare_attention, "probabilities": _prepare_probabilities, "verify_drafts": _prepare_verify,
            "keep_tokens": _prepare_keep}[case["kind"]](case, g, rng)


def _prepare_attention(case, g, rng):
    nh, nkv, d, dtype = case["heads"], case["kv_heads"], case["dim"], DTYPES[case["dtype"]]
    trees, contexts = _lengths(case)
    starts = _starts(trees)
    N, words = starts[-1], (max(trees) + 31) // 32
    table, pages = _tables(g, contexts)
    transposed = dtype == torch.bfloat16        # the engine keeps value pages transposed in bfloat16
    k = torch.randn((pages, nkv, PAGE, d), generator=g, device=DEVICE).to(dtype)
    v = torch.randn((pages, nkv, d, PAGE) if transposed else (pages, nkv, PAGE, d), generator=g, device=DEVICE).to(dtype)
    # the step's queries are the first columns of the joint projection of queries, keys and values
    qkv = (1.5 * torch.randn((N, (nh + 2 * nkv) * d), generator=g, device=DEVICE)).to(dtype)
    parents = [_tree(rng, n, 3) for n in trees]
    depths = []
    for p in parents:
        depth = []
        for x in p:
            depth.append(0 if x < 0 else depth[x] + 1)
        depths.append(depth)
    state = {"case": case, "trees": trees, "contexts": contexts, "starts": starts, "table": table, "k": k, "v": v,
             "transposed": transposed, "q": qkv[:, :nh * d], "scale": d ** -0.5,
             "mask": _ints([w for p in parents for w in _masks(p, words)]).view(N, words),
             "out": torch.empty((N, nh * d), dtype=dtype, device=DEVICE)}
    if own:
        from llm_infrence_engine_amd.parts.base import KVView, StepContext

        R = len(trees)
        rows = _ints(list(range(R)))
        slots = _ints([-1] * N)     # (the step has stored its keys and values already)
        state["kv"] = KVView({"k": k, "v": v}, {"k": False, "v": transposed}, table, slots, table_rows=rows)
        state["ctx"] = StepContext(
            N, R, _ints([0] * N), _ints([c - n + i for c, n, dep in zip(contexts, trees, depths) for i in dep]),
            _ints([r for r, n in enumerate(trees) for _ in range(n)]), _ints(starts), _ints(contexts), rows,
            _ints(list(range(N))), max(trees), max(contexts))
    return state


def _logits(shape, g):
    """Logits whose softmax falls off with the rank's power, as a language model's next-token distributions do; how fast
    differs from row to row."""
    sharp = 1.2 + 0.8 * torch.rand((shape[0], 1), generator=g, device=DEVICE)
    return -sharp * torch.log(1.0 - torch.rand(shape, generator=g, device=DEVICE)) - 5.0


def _prepare_probabilities(case, g, rng):
    M, V = case["rows"], case["vocab"]
    dev = {"dtype": torch.float32, "device": DEVICE}
    return {"case": case, "logits": _logits((M, V), g), "out": torch.empty((M, V), **dev),
            "temperature": torch.full((M,), case["temperature"], **dev),
            "top_k": torch.full((M,), case["top_k"], dtype=torch.int32, device=DEVICE),
            "top_p": torch.full((M,), case["top_p"], **dev)}


def _prepare_verify(case, g, rng):
    R, V, nodes = case["requests"], case["vocab"], case["nodes"]
    trees = [nodes] + [rng.randint((nodes + 1) // 2, nodes) for _ in range(R - 1)]
    starts = _starts(trees)
    N = starts[-1]
    parents = [p for n in trees for p in _tree(rng, n, case["width"])]
    logits = _logits((N, V), g)
    p = torch.softmax(logits, dim=1)
    q = torch.softmax(logits + 0.7 * torch.randn((N, V), generator=g, device=DEVICE), dim=1)     # a draft model's
    # every guess is drawn from its parent's distribution (the root's token is the request's last one)
    first = torch.tensor([starts[r] for r, n in enumerate(trees) for _ in range(n)], device=DEVICE)
    up = first + _ints(parents).long().clamp(min=0)
    guess = torch.multinomial(q, case["width"], replacement=True, generator=g)
    which = torch.randint(0, case["width"], (N,), generator=g, device=DEVICE)
    tokens = guess[up, which].int()
    return {"case": case, "p": p, "q": q if case["drawn"] else None, "tokens": tokens, "parents": _ints(parents),
            "starts": _ints(starts), "uniforms": torch.rand((N,), generator=g, device=DEVICE), "most": max(trees),
            "nodes": torch.empty((R, nodes), dtype=torch.int32, device=DEVICE),
            "counts": torch.empty((R,), dtype=torch.int32, device=DEVICE),
            "next": torch.empty((R,), dtype=torch.int32, device=DEVICE)}


def _prepare_keep(case, g, rng):
    R, L, nkv, d, dtype = case["requests"], case["layers"], case["kv_heads"], case["dim"], DTYPES[case["dtype"]]
    trees, contexts = _lengths(case)
    trees = [case["nodes"]] * R
    contexts = [max(c, case["nodes"]) for c in contexts]
    table, pages = _tables(g, contexts)
    transposed = dtype == torch.bfloat16
    k = torch.randn((L, pages, nkv, PAGE, d), generator=g, device=DEVICE).to(dtype)
    v = torch.randn((L, pages, nkv, d, PAGE) if transposed else (L, pages, nkv, PAGE, d), generator=g, device=DEVICE).to(dtype)
    # the path leaves the root for tokens beyond the places it moves to, so that doing it again changes nothing
    D = case["depth"] + 1
    nodes, counts = [], []
    for _ in range(R):
        count = rng.randint(1, D)
        path = [0] + sorted(rng.sample(range(D, case["nodes"]), count - 1))
        nodes.append(path + [-1] * (D - count))
        counts.append(count)
    return {"case": case, "k": k, "v": v, "transposed": transposed, "table": table,
            "first": _ints([c - n for c, n in zip(contexts, trees)]), "nodes": _ints(nodes), "counts": _ints(counts),
            "rows": _ints(list(range(R)))}


# --------------------------------------------------------------------------------------------------------- one pass
def run(state):
    kind = state["case"]["kind"]
    if own:
        return _run_own(kind, state)
    return {"tree_attention": _plain_attention, "probabilities": _plain_probabilities, "verify_drafts": _plain_verify,
            "keep_tokens": _plain_keep}[kind](state)


def _run_own(kind, s):
    from llm_infrence_engine_amd.kernels import ops

    case = s["case"]
    if kind == "tree_attention":
        return ops.tree_attention(s["q"], s["kv"], s["ctx"], s["mask"], s["out"], case["heads"], s["scale"])
    if kind == "probabilities":
        return ops.probabilities(s["logits"], s["out"], s["temperature"], s["top_k"], s["top_p"],
                                 use_top_k=0 < case["top_k"] < case["vocab"], use_top_p=case["top_p"] < 1.0)
    if kind == "verify_drafts":
        ops.verify_drafts(s["p"], s["q"], s["tokens"], s["parents"], s["starts"], s["uniforms"], s["nodes"], s["counts"], s["next"])
        return s["nodes"], s["counts"], s["next"]
    ops.keep_tokens([s["k"], s["v"]], [False, s["transposed"]], s["table"], s["first"], s["nodes"], s["counts"], s["rows"])
    return s["k"], s["v"]


def _plain_attention(s):
    """out[n, h] = sum over visible j of softmax_j(scale q[n, h] . k_j) v_j, request by request."""
    case = s["case"]
    nh, nkv, d = case["heads"], case["kv_heads"], case["dim"]
    rep = nh // nkv
    for r, (n, c) in enumerate(zip(s["trees"], s["contexts"])):
        t0 = s["starts"][r]
        pages = s["table"][r, :-(-c // PAGE)].long()
        k, v = s["k"][pages].float(), s["v"][pages].float()
        if s["transposed"]:
            v = v.transpose(2, 3)
        k = k.permute(1, 0, 2, 3).reshape(nkv, -1, d)[:, :c]
        v = v.permute(1, 0, 2, 3).reshape(nkv, -1, d)[:, :c].contiguous()
        q = s["q"][t0:t0 + n].float().reshape(n, nkv, rep, d).permute(1, 0, 2, 3).reshape(nkv, n * rep, d)
        scores = torch.matmul(q, k.transpose(1, 2).contiguous()) * s["scale"]
        place = torch.arange(c, device=DEVICE) - (c - n)      # of a key among the step's tokens; below 0: cached before
        at = place.clamp(min=0)
        bits = (s["mask"][t0:t0 + n].long()[:, at // 32] >> (at % 32)) & 1
        sees = (bits != 0) | (place < 0)
        scores = torch.where(sees.repeat_interleave(rep, dim=0), scores, float("-inf"))
        top = scores.amax(dim=2, keepdim=True)
        e = torch.exp(scores - torch.where(torch.isinf(top), torch.zeros_like(top), top))
        total = e.sum(dim=2, keepdim=True)
        o = torch.matmul(e, v) / torch.where(total > 0, total, torch.ones_like(total))
        s["out"][t0:t0 + n] = o.reshape(nkv, n, rep, d).permute(1, 0, 2, 3).reshape(n, nh * d).to(s["out"].dtype)
    return s["out"]


def _plain_probabilities(s):
    """softmax(logits / T) over the tokens kept: the k largest (with ties), of these the smallest set of the largest whose
    mass reaches p (with ties)."""
    case = s["case"]
    x = s["logits"] * (1.0 / s["temperature"])[:, None]
    if 0 < case["top_k"] < case["vocab"]:
        kth = torch.topk(x, case["top_k"], dim=1).values[:, -1:]
        x = torch.where(x >= kth, x, float("-inf"))
    top = x.amax(dim=1, keepdim=True)
    if case["top_p"] < 1.0:
        ordered = torch.sort(x, dim=1, descending=True).values
        e = torch.exp((ordered - top).double())
        before = torch.cumsum(e, dim=1) - e
        kept = before < s["top_p"][:, None].double() * e.sum(dim=1, keepdim=True)
        least = torch.where(kept, ordered, float("inf")).amin(dim=1, keepdim=True)
        x = torch.where(x >= least, x, float("-inf"))
    e = torch.exp(x - top)
    s["out"].copy_(e / e.sum(dim=1, keepdim=True))
    return s["out"]


def _plain_verify(s):
    """Every request's tree at once, token after token: a token is looked at when its parent is the last one accepted.

    Guess x behind a token with target p and draft q: accepted if u q(x) S < p(x) - t q(x), where t and S start at 0 and 1;
    if it is not, t becomes t + S and S the sum of max(0, p - t q).  A guess without a distribution stands for itself: q is
    1 there, and p loses the guesses that were not accepted.  Behind the last one accepted a token is drawn from
    max(0, p - t q) with the root's number.
    """
    case, p, q = s["case"], s["p"], s["q"]
    R, V, most = case["requests"], case["vocab"], s["most"]
    starts = s["starts"].long()
    first, length = starts[:-1], starts[1:] - starts[:-1]
    each = torch.arange(R, device=DEVICE)
    at = torch.zeros(R, dtype=torch.long, device=DEVICE)
    t = torch.zeros(R, dtype=torch.float64, device=DEVICE)
    S = torch.ones(R, dtype=torch.float64, device=DEVICE)
    gone = torch.zeros((R, V), dtype=torch.bool, device=DEVICE) if q is None else None
    nodes = torch.full((R, case["nodes"]), -1, dtype=torch.long, device=DEVICE)
    nodes[:, 0] = 0
    counts = torch.ones(R, dtype=torch.long, device=DEVICE)
    for i in range(1, most):
        n = first + torch.clamp(torch.full_like(first, i), max=length - 1)
        child = (i < length) & (s["parents"][n] == at)
        x = s["tokens"][n].long()
        u = s["uniforms"][n].double()
        px = p[first + at, x].double()
        if q is None:
            px = torch.where(gone[each, x], torch.zeros_like(px), px)
            taken = child & (u * S < px)
        else:
            qx = q[first + at, x].double()
            taken = child & (u * qx * S < px - t * qx)
        refused = child & ~taken
        if q is None:
            S = torch.where(refused, S - px, S)
            gone[each, x] |= refused
        else:
            t = torch.where(refused, t + S, t)
            S = torch.where(refused, (p[first + at].double() - t[:, None] * q[first + at].double()).clamp(min=0).sum(dim=1), S)
        at = torch.where(taken, torch.full_like(at, i), at)
        t = torch.where(taken, torch.zeros_like(t), t)
        S = torch.where(taken, torch.ones_like(S), S)
        if q is None:
            gone &= ~taken[:, None]
        place = torch.clamp(counts, max=case["nodes"] - 1)
        nodes[each, place] = torch.where(taken, torch.full_like(at, i), nodes[each, place])
        counts = counts + taken.long()
    rest = p[first + at].double()
    whole = rest
    rest = torch.where(gone, torch.zeros_like(rest), rest) if q is None else (rest - t[:, None] * q[first + at].double()).clamp(min=0)
    rest = torch.where(rest.sum(dim=1, keepdim=True) > 0, rest, whole)
    run_ = torch.cumsum(rest, dim=1)
    drawn = (run_ > s["uniforms"][first].double()[:, None] * run_[:, -1:]).to(torch.int32).argmax(dim=1)
    s["nodes"].copy_(nodes)
    s["counts"].copy_(counts)
    s["next"].copy_(drawn)
    return s["nodes"], s["counts"], s["next"]


def _plain_keep(s):
    """The entry of the path's i-th token to the i-th place behind the cached ones, in every layer."""
    R, D = s["nodes"].shape
    i = torch.arange(D, device=DEVICE)[None, :]
    valid = i < s["counts"][:, None]
    to = s["first"][:, None].long() + i
    of = torch.where(valid, s["first"][:, None].long() + s["nodes"].long(), to)
    # (places beyond the path are written with what they hold)
    each = torch.arange(R, device=DEVICE)[:, None]
    of_page, of_slot = s["table"][each, of // PAGE].long(), of % PAGE
    to_page, to_slot = s["table"][each, to // PAGE].long(), to % PAGE
    for pages, transposed in ((s["k"], False), (s["v"], s["transposed"])):
        if transposed:
            pages[:, to_page, :, :, to_slot] = pages[:, of_page, :, :, of_slot]
        else:
            pages[:, to_page, :, to_slot] = pages[:, of_page, :, of_slot]
    return s["k"], s["v"]


# --------------------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"tree_attention": _exact_attention, "probabilities": _exact_probabilities, "verify_drafts": _exact_verify,
            "keep_tokens": _exact_keep}[case["kind"]](s)


def _exact_attention(s):
    case = s["case"]
    nh, nkv, d = case["heads"], case["kv_heads"], case["dim"]
    out = torch.zeros((s["starts"][-1], nh, d), dtype=torch.float64, device=DEVICE)
    for r, (n, c) in enumerate(zip(s["trees"], s["contexts"])):
        t0 = s["starts"][r]
        place = torch.arange(c, device=DEVICE)
        page, slot = s["table"][r].long()[place // PAGE], place % PAGE
        hidden = torch.zeros((n, c), dtype=torch.bool, device=DEVICE)
        for i, words in enumerate(s["mask"][t0:t0 + n].tolist()):
            bits = sum((w & 0xFFFFFFFF) << (32 * j) for j, w in enumerate(words))
            hidden[i, c - n:] = torch.tensor([not (bits >> j) & 1 for j in range(n)], device=DEVICE)
        for h in range(nh):
            g = h // (nh // nkv)
            k = s["k"][page, g, slot].double()
            v = (s["v"][page, g, :, slot] if s["transposed"] else s["v"][page, g, slot]).double()
            q = s["q"][t0:t0 + n, h * d:(h + 1) * d].double()
            scores = (q @ k.t().contiguous()) * s["scale"]
            scores[hidden] = -math.inf
            out[t0:t0 + n, h] = torch.softmax(scores, dim=1) @ v      # (every token of these trees sees itself)
    return out.view(-1, nh * d)


def _exact_probabilities(s):
    case = s["case"]
    out = torch.zeros((case["rows"], case["vocab"]), dtype=torch.float64, device=DEVICE)
    for r in range(case["rows"]):
        x = s["logits"][r].double() / s["temperature"][r].double()
        order = torch.argsort(x, descending=True)
        n = case["top_k"] if 0 < case["top_k"] < case["vocab"] else case["vocab"]
        x = x[order]
        w = torch.exp(x - x[0])
        w[x < x[n - 1]] = 0.0
        if case["top_p"] < 1.0:
            upto = torch.cumsum(w, dim=0)
            last = int(torch.searchsorted(upto, s["top_p"][r].double() * upto[-1]))     # the first whose sum reaches it
            w[x < x[last]] = 0.0
        out[r, order] = w / w.sum()
    return out


def _exact_verify(s):
    case = s["case"]
    R = case["requests"]
    starts, parents, tokens = s["starts"].tolist(), s["parents"].tolist(), s["tokens"].tolist()
    u = s["uniforms"].double().tolist()
    nodes = torch.full((R, case["nodes"]), -1, dtype=torch.int32)
    counts, drawn = [], []
    for r in range(R):
        base, length = starts[r], starts[r + 1] - starts[r]
        path = [0]
        while True:
            here = path[-1]
            p = s["p"][base + here].double()
            rest, mass = p.clone(), 1.0       # what is left of the target behind the guesses refused so far
            draft = None if s["q"] is None else s["q"][base + here].double()
            weight, taken = 0.0, None
            for i in range(here + 1, length):
                if parents[base + i] != here:
                    continue
                x = tokens[base + i]
                if draft is None:
                    ok = u[base + i] * mass < float(rest[x])
                else:
                    ok = u[base + i] * float(draft[x]) * mass < float(p[x]) - weight * float(draft[x])
                if ok:
                    taken = i
                    break
                if draft is None:
                    mass -= float(rest[x])
                    rest[x] = 0.0
                else:
                    weight += mass
                    rest = (p - weight * draft).clamp(min=0.0)
                    mass = float(rest.sum())
            if taken is None:
                break
            path.append(taken)
        rest = rest if float(rest.sum()) > 0 else p
        upto = torch.cumsum(rest, dim=0)
        drawn.append(int(torch.nonzero(upto > u[base] * float(upto[-1]))[0]))
        nodes[r, :len(path)] = torch.tensor(path, dtype=torch.int32)
        counts.append(len(path))
    return nodes.to(DEVICE), _ints(counts), _ints(drawn)


def _exact_keep(s):
    table, first, counts = s["table"].tolist(), s["first"].tolist(), s["counts"].tolist()
    for r, path in enumerate(s["nodes"].tolist()):
        for i, n in enumerate(path[:counts[r]]):
            a, b = first[r] + n, first[r] + i
            ap, as_, bp, bs = table[r][a // PAGE], a % PAGE, table[r][b // PAGE], b % PAGE
            s["k"][:, bp, :, bs] = s["k"][:, ap, :, as_]
            if s["transposed"]:
                s["v"][:, bp, :, :, bs] = s["v"][:, ap, :, :, as_]
            else:
                s["v"][:, bp, :, bs] = s["v"][:, ap, :, as_]
    return s["k"], s["v"]
