"""The operators of a step that checks trees of drafted tokens: each alone against a plain implementation in 64 bits, what they
refuse, and a step of them together."""
import math
import random
from types import SimpleNamespace

import pytest
import torch

from llm_infrence_engine_amd.kernels import ops

DEV = "cuda:0"
gpu = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def ints(values, device=DEV):
    return torch.tensor(values, dtype=torch.int32, device=device)


def random_tree(rng, n, width=3):
    """Parents; a child comes after its parent."""
    return [-1] + [rng.randint(max(0, i - 1 - width), i - 1) for i in range(1, n)]


def ancestors(parents):
    sees = []
    for n, p in enumerate(parents):
        sees.append((sees[p] if p >= 0 else set()) | {n})
    return sees


def mask_words(sees, words):
    rows = []
    for s in sees:
        row = [0] * words
        for j in s:
            row[j // 32] |= 1 << (j % 32)
        rows.append([w - (1 << 32) if w >= 1 << 31 else w for w in row])
    return rows


# ------------------------------------------------------------------------------------------------ attention
def make_step(dtype, nh, nkv, d, page_size, trees, contexts, *, dv=None, transposed=None, seed=0, words=None, sees=None, extra_cols=8,
              q_scale=1.5, max_context=None):
    """A step over pages in scrambled order whose unused places hold NaN; ``sees[r][i]``: the tokens that token i of request r
    sees (default: its ancestors in a random tree)."""
    g = torch.Generator().manual_seed(seed)
    rng = random.Random(seed)
    dv = dv or d
    R, N = len(trees), sum(trees)
    if transposed is None:
        transposed = dtype == BF16 and page_size % 16 == 0
    sees = sees or [ancestors(random_tree(rng, n)[:n]) for n in trees]
    words = words or max(1, (max(trees + [1]) + 31) // 32)
    need = [-(-c // page_size) for c in contexts]
    order = list(range(1, sum(need) + 3))
    rng.shuffle(order)
    rows = list(range(R + 2))
    rng.shuffle(rows)
    rows = rows[:R]
    table = torch.zeros(R + 2, max(need + [1]) + 2, dtype=torch.int32)
    K = [torch.randn(nkv, c, d, generator=g).to(dtype) for c in contexts]
    V = [torch.randn(nkv, c, dv, generator=g).to(dtype) for c in contexts]
    P = sum(need) + 3
    k = torch.full((P, nkv, page_size, d), math.nan).to(dtype)
    v = torch.full((P, nkv, page_size, dv), math.nan).to(dtype)
    for r, c in enumerate(contexts):
        for b in range(need[r]):
            page = order.pop()
            table[rows[r], b] = page
            part = slice(b * page_size, min(c, (b + 1) * page_size))
            k[page, :, :part.stop - part.start] = K[r][:, part]
            v[page, :, :part.stop - part.start] = V[r][:, part]
    q = (q_scale * torch.randn(N, nh * d + extra_cols, generator=g)).to(dtype)
    starts = [0]
    for n in trees:
        starts.append(starts[-1] + n)
    tree = torch.tensor([w for s in sees for w in mask_words(s, words)], dtype=torch.int32).view(N, words) if N else \
        torch.zeros(0, words, dtype=torch.int32)
    kv = SimpleNamespace(k_pages=k.to(DEV), v_pages=(v.transpose(2, 3).contiguous() if transposed else v).to(DEV), v_transposed=transposed,
                         block_table=table.to(DEV), table_rows=ints(rows))
    ctx = SimpleNamespace(token_req=ints([r for r, n in enumerate(trees) for _ in range(n)]), q_start=ints(starts),
                          context_lens=ints(contexts), max_q_len=max(trees + [1]), max_context_len=max_context or max(contexts + [1]),
                          n_live_tokens=None)
    return SimpleNamespace(q=q.to(DEV)[:, :nh * d], kv=kv, ctx=ctx, tree=tree.to(DEV), K=K, V=V, sees=sees, starts=starts, trees=trees,
                           contexts=contexts, nh=nh, nkv=nkv, d=d, dv=dv, scale=d ** -0.5, dtype=dtype,
                           out=torch.full((N, nh * dv), 7.0, device=DEV).to(dtype))


def plain_attention(s):
    """(result, sum of the weights times |values|), float64 [N, nh, dv]; keys that are not visible are left out, not weighted."""
    N = s.starts[-1]
    want, size = (torch.zeros(N, s.nh, s.dv, dtype=torch.float64) for _ in range(2))
    q = s.q.cpu().double().view(N, s.nh, s.d)
    for r, (n, c) in enumerate(zip(s.trees, s.contexts)):
        for i in range(n):
            keys = list(range(c - n)) + [c - n + j for j in sorted(s.sees[r][i]) if j < n]
            if not keys:
                continue
            for g in range(s.nkv):
                k, v = s.K[r][g, keys].double(), s.V[r][g, keys].double()
                heads = slice(g * (s.nh // s.nkv), (g + 1) * (s.nh // s.nkv))
                w = torch.softmax(q[s.starts[r] + i, heads] @ k.t() * s.scale, dim=-1)
                want[s.starts[r] + i, heads] = w @ v
                size[s.starts[r] + i, heads] = w @ v.abs()
    return want, size


def close_enough(s, got=None):
    """bfloat16: the probabilities and the result are rounded once each, 2^-8 relative at most: the sum of weighted values is off
    by 2^-8 of that of their magnitudes, its denominator by 2^-8, the result by 2^-8.  float: a score is a sum of d products,
    each rounded by 2^-24 of about 10, sqrt(d) of which add up (d = 256: 1e-5), as do the weighted values."""
    want, size = plain_attention(s)
    got = (s.out if got is None else got).cpu().double().view(want.shape)
    e = 2.0 ** -8 if s.dtype == BF16 else 0.0
    limit = 2e-5 + (4e-5 if s.dtype == BF16 else 0.0) + e * (size + 2 * want.abs())
    off = (got - want).abs()
    bad = ~(off <= limit)
    assert not bad.any(), (int(bad.sum()), off[bad].max(), bad.nonzero()[:4].tolist())


ATTENTION = [
    # nh, nkv, d, page size, trees, contexts
    (14, 2, 64, 16, [8], [200]),
    (14, 2, 64, 16, [1], [1]),                                   # one token that sees itself
    (7, 1, 64, 16, [1, 1, 1], [1, 2, 65]),
    (14, 2, 64, 16, [5, 0, 3, 1], [5, 0, 70, 64]),               # nothing cached before, a request without tokens
    (28, 4, 128, 16, [16, 9, 13], [300, 700, 129]),
    (40, 8, 128, 16, [63, 2], [1000, 2]),
    (6, 2, 32, 16, [33, 32, 31], [33, 96, 512]),
    (4, 4, 128, 32, [64, 65], [64, 190]),                        # trees on both sides of two words
    (4, 2, 64, 48, [100], [333]),
    (8, 1, 64, 64, [150], [400]),
    (32, 1, 128, 16, [3, 7], [90, 31]),                          # a group of 32
    (5, 1, 48, 16, [9, 4], [70, 33]),                            # sizes of the kernel for any
    (4, 2, 20, 7, [9, 4], [70, 33]),
    (2, 1, 256, 16, [3], [20]),
    (3, 3, 64, 4, [12], [77]),
]


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("case", range(len(ATTENTION)))
def test_tree_attention(dtype, case):
    s = make_step(dtype, *ATTENTION[case], seed=case)
    ops.tree_attention(s.q, s.kv, s.ctx, s.tree, s.out, s.nh, s.scale)
    close_enough(s)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("nh,nkv,d", [(14, 2, 64), (8, 2, 128), (4, 2, 32)])
def test_tree_attention_of_long_contexts(dtype, nh, nkv, d):
    s = make_step(dtype, nh, nkv, d, 16, [12, 3, 1], [3001, 1100, 4096], seed=5)
    ops.tree_attention(s.q, s.kv, s.ctx, s.tree, s.out, s.nh, s.scale)
    close_enough(s)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_tree_attention_layouts(dtype):
    """Values as they are stored in both layouts, values of another size than keys, rows that begin anywhere, without table rows."""
    for kw in ({"transposed": False}, {"transposed": True}, {"dv": 32}, {"extra_cols": 1}, {"extra_cols": 3}, {"words": 4}):
        s = make_step(dtype, 8, 2, 64, 16, [9, 17], [50, 130], seed=3, **kw)
        ops.tree_attention(s.q, s.kv, s.ctx, s.tree, s.out, s.nh, s.scale)
        close_enough(s)
    s = make_step(dtype, 8, 2, 64, 16, [9, 17], [50, 130], seed=3)
    s.kv.block_table = s.kv.block_table[s.kv.table_rows.long()].contiguous()
    s.kv.table_rows = None
    ops.tree_attention(s.q, s.kv, s.ctx, s.tree, s.out, s.nh, s.scale)
    close_enough(s)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("nh,nkv,d", [(14, 2, 64), (8, 2, 128), (4, 2, 32)])
def test_tree_attention_masks(dtype, nh, nkv, d):
    """Rows that see nothing get zeros; bits behind the tree count for nothing; any set of tokens may be visible."""
    rng = random.Random(1)
    trees, contexts = [40, 20, 6], [40, 31, 400]
    sees = [[{j for j in range(n) if rng.random() < 0.4} for _ in range(n)] for n in trees]
    sees[0][0], sees[0][17], sees[0][39], sees[1][3] = set(), set(), set(), set()
    sees[0][5] = set(range(40))
    sees[2][1] = set()
    sees[1][4] = {0, 7, 19} | {25, 31, 40, 63}
    s = make_step(dtype, nh, nkv, d, 16, trees, contexts, seed=2, sees=sees, words=2)
    ops.tree_attention(s.q, s.kv, s.ctx, s.tree, s.out, s.nh, s.scale)
    close_enough(s)
    assert (s.out.view(-1, nh * d)[[0, 17, 39]] == 0).all() and not (s.out[41:42] == 0).all()


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("nh,nkv,d", [(14, 2, 64), (8, 2, 128), (4, 2, 32), (6, 1, 20)])
def test_tree_attention_keeps_what_is_not_visible_out(dtype, bad, nh, nkv, d):
    """A token whose key or value is not finite spoils the results of those that see it, and no others."""
    rng = random.Random(4)
    trees, contexts = [37, 9, 24], [52, 9, 300]
    sees = [ancestors(random_tree(rng, n)) for n in trees]
    s = make_step(dtype, nh, nkv, d, 16, trees, contexts, seed=6, sees=sees)
    spoiled = {(0, 11), (0, 36), (1, 4), (2, 13)}
    clean = SimpleNamespace(**vars(s))
    for which in ("k_pages", "v_pages"):
        pages = getattr(s.kv, which)
        hurt = pages.clone()
        for r, i in spoiled:
            at = contexts[r] - trees[r] + i
            page, slot = int(s.kv.block_table[s.kv.table_rows[r], at // 16]), at % 16
            if which == "v_pages" and s.kv.v_transposed:
                hurt[page, :, :, slot] = bad
            else:
                hurt[page, :, slot] = bad
        setattr(s.kv, which, hurt)
        ops.tree_attention(s.q, s.kv, s.ctx, s.tree, s.out, s.nh, s.scale)
        setattr(s.kv, which, pages)
        want, size = plain_attention(clean)
        got = s.out.cpu().double().view(want.shape)
        e = 2.0 ** -8 if dtype == BF16 else 0.0
        for r, n in enumerate(trees):
            for i in range(n):
                row = s.starts[r] + i
                if any((r, j) in spoiled for j in sees[r][i]):
                    if which == "v_pages":
                        assert not torch.isfinite(got[row]).any(), (which, r, i)
                else:
                    off = (got[row] - want[row]).abs()
                    assert (off <= 6e-5 + e * (size[row] + 2 * want[row].abs())).all(), (which, r, i, off.max())


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_tree_attention_of_a_padded_batch(dtype):
    """Tokens from n_live_tokens on are left as they are, requests without tokens cost nothing, bounds may be loose."""
    s = make_step(dtype, 14, 2, 64, 16, [5, 7, 0, 0], [40, 90, 0, 0], seed=9)
    N = 12
    pad = torch.zeros(16, 14 * 64, dtype=dtype, device=DEV)
    pad[:N] = s.q
    out = torch.full((16, 14 * 64), 3.0, device=DEV).to(dtype)
    tree = torch.zeros(16, 2, dtype=torch.int32, device=DEV)
    tree[:N, :1] = s.tree
    s.ctx.token_req = torch.cat([s.ctx.token_req, ints([0] * 4)])
    s.ctx.n_live_tokens = ints([N])
    s.ctx.max_q_len, s.ctx.max_context_len = 16, 96
    ops.tree_attention(pad, s.kv, s.ctx, tree, out, 14, s.scale)
    close_enough(s, out[:N])
    assert (out[N:] == 3.0).all()


@gpu
@pytest.mark.parametrize("nh,nkv,d", [(14, 2, 64), (8, 2, 128), (4, 2, 32)])
@pytest.mark.parametrize("kind", range(4))
def test_tree_attention_of_every_kind_of_block(monkeypatch, nh, nkv, d, kind):
    """Whatever kind of block and share of the keys a step's sizes ask for: 64 to 4,096 keys a block, some blocks without any."""
    get = ops._get
    for share in (64, 192, 448, 4096):
        monkeypatch.setattr(ops, "_get", lambda name: (lambda *a: kind * 65536 + share // 64) if name == "ms_tree_attention_mfma_plan" else get(name))
        s = make_step(BF16, nh, nkv, d, 16, [12, 0, 37, 1], [1301, 0, 75, 640], seed=7)
        ops.tree_attention(s.q, s.kv, s.ctx, s.tree, s.out, s.nh, s.scale)
        close_enough(s)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("d", [64, 48])
def test_tree_attention_of_tokens_that_are_nobodys(dtype, d):
    """Tokens behind the last request's stay as they are without a count of live ones too."""
    s = make_step(dtype, 8, 2, d, 16, [5, 7], [40, 90], seed=9)
    N = 12
    pad, out = torch.zeros(15, 8 * d, dtype=dtype, device=DEV), torch.full((15, 8 * d), 3.0, device=DEV).to(dtype)
    pad[:N] = s.q
    tree = torch.full((15, 1), -1, dtype=torch.int32, device=DEV)
    tree[:N] = s.tree
    s.ctx.token_req = torch.cat([s.ctx.token_req, ints([0, 1, 1])])
    ops.tree_attention(pad, s.kv, s.ctx, tree, out, 8, s.scale)
    close_enough(s, out[:N])
    assert (out[N:] == 3.0).all()


@gpu
@pytest.mark.parametrize("nh,nkv,d", [(14, 2, 64), (8, 2, 128), (4, 2, 32)])
@pytest.mark.parametrize("share", [64, 192, 4096])
def test_tree_attention_weights_are_not_rounded_to_bfloat16(monkeypatch, nh, nkv, d, share):
    """The result is off by its own rounding, 2^-8 of itself, and hardly more: the weights come in two parts that are off by 2^-15 of
    a weight together, in the sum of weighted values as in the one that divides (2^-14 of both, second-order terms with it), and
    scores, exponentials and sums are floats, as the limits of ``close_enough`` have them."""
    get = ops._get
    for kind in range(4):
        monkeypatch.setattr(ops, "_get", lambda name: (lambda *a: kind * 65536 + share // 64) if name == "ms_tree_attention_mfma_plan" else get(name))
        s = make_step(BF16, nh, nkv, d, 16, [12, 0, 37, 1], [1301, 0, 75, 640], seed=7)
        ops.tree_attention(s.q, s.kv, s.ctx, s.tree, s.out, s.nh, s.scale)
        want, size = plain_attention(s)
        off = (s.out.cpu().double().view(want.shape) - want).abs()
        assert (off <= 6e-5 + 2.0 ** -8 * want.abs() + 2.0 ** -14 * (size + want.abs())).all(), (kind, off.max())


@gpu
@pytest.mark.parametrize("trees,contexts", [([7, 4], [49, 60]), ([2, 3, 5], [34, 48, 60])])
def test_tree_attention_sums_scores_of_floats_in_short_chains(trees, contexts):
    """Roundings that are independent of each other, each half a step over sqrt(3): a score of 128 dims in four chains of 32 sums of up
    to 8 (half a step 2.4e-7) is off by 2.4e-7 / sqrt(3) * sqrt(128) * 0.6 = 9.4e-7, times the scale 0.8e-7; the exponent, up to 8 in
    powers of two, by 1e-7; the exponential 0.7e-7, sums and quotient 0.6e-7: 1.6e-7 together, of a weight and so of a result of
    random values.  Twice that is allowed; one chain of 128 sums of up to 16 had 4.5e-7."""
    s = make_step(F32, 8, 2, 128, 16, trees, contexts, seed=3)
    ops.tree_attention(s.q, s.kv, s.ctx, s.tree, s.out, s.nh, s.scale)
    want, _ = plain_attention(s)
    off = (s.out.cpu().double().view(want.shape) - want).norm() / want.norm()
    assert off <= 3.2e-7, off


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("bad", [math.inf, -math.inf])
@pytest.mark.parametrize("nh,nkv,d", [(14, 2, 64), (8, 2, 128), (4, 2, 32), (6, 1, 20)])
def test_tree_attention_of_infinite_values(monkeypatch, dtype, bad, nh, nkv, d):
    """A visible value that is infinite makes the result infinite, not NaN, however the keys are shared out (every weight is far from
    underflow: a score is 1.5 times a normal number); one cached before the step does so for all."""
    get = ops._get
    trees, contexts = [9, 24], [640, 1170]
    sees = [ancestors(random_tree(random.Random(4), n)) for n in trees]
    for share in (128, 256, 384, 2048):
        forced = {"ms_tree_attention_mfma_plan": 2 * 65536 + share // 64, "ms_tree_attention_f32_share": share}
        monkeypatch.setattr(ops, "_get", lambda name: (lambda *a: forced[name]) if name in forced else get(name))
        for at, seen in ((contexts[1] - trees[1] + 13, [i for i in range(24) if 13 in sees[1][i]]), (70, range(24))):
            s = make_step(dtype, nh, nkv, d, 16, trees, contexts, seed=6, sees=sees)
            page, slot = int(s.kv.block_table[s.kv.table_rows[1], at // 16]), at % 16
            if s.kv.v_transposed:
                s.kv.v_pages[page, :, :, slot] = bad
            else:
                s.kv.v_pages[page, :, slot] = bad
            ops.tree_attention(s.q, s.kv, s.ctx, s.tree, s.out, s.nh, s.scale)
            got = s.out.cpu().float()
            for n in range(s.starts[-1]):
                hit = n >= 9 and n - 9 in seen
                assert (got[n] == bad).all() if hit else torch.isfinite(got[n]).all(), (share, at, n)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("nh,nkv,d", [(4, 2, 64), (2, 1, 128), (4, 2, 32)])
def test_tree_attention_of_more_than_64_shares(monkeypatch, dtype, nh, nkv, d):
    """The join has a second part for a lane from the 65th share on; what stands in those decides the result: the step's own values
    are a hundred times the others.  The two parts with their sums are floats: nothing on top of ``close_enough``."""
    get = ops._get
    for share in (128, 192):
        forced = {"ms_tree_attention_mfma_plan": 65536 + share // 64, "ms_tree_attention_f32_share": share}
        monkeypatch.setattr(ops, "_get", lambda name: (lambda *a: forced[name]) if name in forced else get(name))
        s = make_step(dtype, nh, nkv, d, 16, [3, 1, 7], [12500, 70 * share + 5, 8400], seed=8)
        for r in range(3):
            for at in range(s.contexts[r] - s.trees[r], s.contexts[r]):
                page, slot = int(s.kv.block_table[s.kv.table_rows[r], at // 16]), at % 16
                s.V[r][:, at] *= 100
                value = s.V[r][:, at].to(DEV)
                if s.kv.v_transposed:
                    s.kv.v_pages[page, :, :, slot] = value
                else:
                    s.kv.v_pages[page, :, slot] = value
        ops.tree_attention(s.q, s.kv, s.ctx, s.tree, s.out, s.nh, s.scale)
        close_enough(s)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("nh,nkv,d", [(14, 2, 64), (8, 2, 128), (4, 2, 32), (6, 1, 20)])
def test_tree_attention_of_a_key_that_is_nan(dtype, nh, nkv, d):
    """A token that sees it gets NaN throughout, one that does not what it gets without."""
    trees, contexts = [37, 9], [300, 9]
    sees = [ancestors(random_tree(random.Random(4), n)) for n in trees]
    s = make_step(dtype, nh, nkv, d, 16, trees, contexts, seed=6, sees=sees)
    at = contexts[0] - trees[0] + 11
    s.kv.k_pages[int(s.kv.block_table[s.kv.table_rows[0], at // 16]), :, at % 16] = math.nan
    ops.tree_attention(s.q, s.kv, s.ctx, s.tree, s.out, s.nh, s.scale)
    for n, row in enumerate(s.out.cpu()):
        hit = n < 37 and 11 in sees[0][n]
        assert torch.isnan(row).all() if hit else torch.isfinite(row).all(), n


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("nh,nkv,d", [(14, 2, 64), (8, 2, 128), (5, 1, 48)])
def test_tree_attention_replayed_with_the_bounds_of_a_cache(dtype, nh, nkv, d):
    """A captured step's bounds are its batch's tokens and the cache's capacity; contexts, trees and the count of live tokens change
    between the replays, each checked against 64 bits and against the eager call."""
    s = make_step(dtype, nh, nkv, d, 16, [8, 5, 13], [300, 40, 2000], seed=1)
    N, R = 32, 3
    table = torch.zeros(s.kv.block_table.shape[0], 2048, dtype=torch.int32, device=DEV)
    table[:, :s.kv.block_table.shape[1]] = s.kv.block_table
    s.kv.block_table = table
    s.ctx.max_q_len, s.ctx.max_context_len = N, 32768
    q, out = torch.zeros(N, nh * d, dtype=dtype, device=DEV), torch.zeros(N, nh * d, dtype=dtype, device=DEV)
    tree, s.ctx.n_live_tokens = torch.zeros(N, 1, dtype=torch.int32, device=DEV), ints([26])
    s.ctx.token_req, s.ctx.q_start, s.ctx.context_lens = ints([0] * N), ints([0] * (R + 1)), ints([0] * R)
    q[:26] = s.q

    def step():
        ops.tree_attention(q, s.kv, s.ctx, tree, out, nh, s.scale)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.inference_mode(), torch.cuda.graph(graph, stream=side):
        step()
    for trees, contexts in (([8, 5, 13], [300, 40, 2000]), ([1, 0, 25], [7, 0, 1999]), ([10, 1, 2], [10, 33, 64]), ([0, 0, 0], [0, 0, 0])):
        sees = [ancestors(random_tree(random.Random(n), n)[:n]) for n in trees]
        starts = [0, trees[0], trees[0] + trees[1], sum(trees)]
        live = starts[-1]
        s.ctx.token_req.copy_(ints([r for r, n in enumerate(trees) for _ in range(n)] + [0] * (N - live)))
        s.ctx.q_start.copy_(ints(starts))
        s.ctx.context_lens.copy_(ints(contexts))
        s.ctx.n_live_tokens.copy_(ints([live]))
        tree.zero_()
        if live:
            tree[:live] = ints([w for x in sees for w in mask_words(x, 1)])
        both = []
        for run in (graph.replay, step):
            out.fill_(3.0)
            run()
            torch.cuda.synchronize()
            both.append(out.clone())
        assert torch.equal(*both) and (out[live:] == 3.0).all()
        now = SimpleNamespace(**{**vars(s), "trees": trees, "contexts": contexts, "sees": sees, "starts": starts, "q": q[:live], "out": out[:live]})
        if live:
            close_enough(now)


# ------------------------------------------------------------------------------------------------ probabilities
def plain_probabilities(logits, T, top_k, top_p):
    """float64, row by row; the scaled logits are floats, as the sampler has them."""
    out = torch.zeros(logits.shape, dtype=torch.float64)
    for r in range(logits.shape[0]):
        x = logits[r]
        t = float(T[r]) if T is not None else 0.0
        if not t > 0:
            y = torch.where(torch.isnan(x), torch.tensor(-math.inf), x)
            out[r, int((y == y.max()).nonzero()[0]) if (y > -math.inf).any() else 0] = 1.0
            continue
        x = (x * (torch.tensor(1.0) / T[r])).double()
        ok = ~torch.isnan(x)
        x = torch.where(ok, x, torch.tensor(-math.inf, dtype=torch.float64))
        if not torch.isfinite(x.max()):
            inf = (x == math.inf)
            out[r, int(inf.nonzero()[0]) if inf.any() else 0] = 1.0
            continue
        k = int(top_k[r]) if top_k is not None else 0
        if 0 < k < x.numel():
            x = torch.where(x >= torch.topk(x, k).values[-1], x, torch.tensor(-math.inf, dtype=torch.float64))
        w = torch.exp(x - x.max())
        p = float(top_p[r]) if top_p is not None else 1.0
        if p < 1.0:
            order = torch.argsort(x, descending=True)
            upto = torch.cumsum(w[order], 0)
            last = int((upto >= p * upto[-1]).nonzero()[0]) if p > 0 else 0
            w = torch.where(x >= x[order[last]], w, torch.zeros_like(w))
        out[r] = w / w.sum()
    return out


def check_probabilities(logits, T, top_k, top_p, **kw):
    """The scaled logits are given as floats; their difference to the maximum is rounded by 2^-24 of at most 40, the exponential by
    a few units and the quotient by one: 40 * 2^-24 + 4 * 2^-24 = 2.7e-6 relative.  The sum's terms are cut at 2^-44 of the
    largest: at most 152,064 * 2^-44 = 1e-8 of it."""
    out = torch.full(logits.shape, 7.0, device=DEV)
    to = lambda t: None if t is None else t.to(DEV)     # noqa: E731
    ops.probabilities(logits.to(DEV), out, to(T), to(top_k), to(top_p), **kw)
    got, want = out.cpu().double(), plain_probabilities(logits, T, top_k, top_p)
    tiny = want < 1e-30     # (exponentials below the floats' range may be none)
    assert ((got > 0) == (want > 0))[~tiny].all(), ((got > 0) != (want > 0)).nonzero()[:5]
    assert (got[tiny] <= 1e-29).all()
    assert ((got - want).abs() <= 2.8e-6 * want)[~tiny].all(), ((got - want).abs() / want)[~tiny].max()


@gpu
@pytest.mark.parametrize("V", [1, 7, 1000, 2049, 40001, 151936])
@pytest.mark.parametrize("T,k,p", [(0.8, 50, 0.9), (1.3, 0, 0.7), (1.0, 5, 1.0), (1.0, 0, 1.0), (0.5, 700, 0.99), (0.7, 1, 0.2), (1.0, 0, 1e-9)])
def test_probabilities(V, T, k, p):
    g = torch.Generator().manual_seed(V)
    M = 3 if V > 50000 else 9
    logits = -1.5 * torch.log(1 - torch.rand(M, V, generator=g)) - 4
    check_probabilities(logits, torch.full((M,), T), ints([k] * M, "cpu"), torch.full((M,), p))


@gpu
def test_probabilities_of_mixed_rows():
    """Every row its own parameters: greedy ones (the first of equal maxima), a k at and beyond the vocabulary, ties at the k-th
    value and at the mass, values of the type's lowest, infinities, NaN, one token alone; rows of many requests."""
    g = torch.Generator().manual_seed(3)
    V = 5000
    logits = 2 * torch.randn(16, V, generator=g)
    logits[1, [40, 7, 4999]] = 30.0                          # equal maxima
    logits[2, 100:110] = logits[2].max() + 1                 # ten alike, k = 4: all stay
    logits[3, :] = 1.5                                       # all alike
    logits[4, 50:] = torch.finfo(F32).min
    logits[5, 50:] = -math.inf
    logits[6, ::3] = math.nan
    logits[7, :] = math.nan
    logits[8, :] = -math.inf
    logits[9, 123] = math.inf
    logits[10, 5:] = -math.inf
    logits[11, 0] = 90.0                                     # everything on one
    T = torch.tensor([0.8, 0.0, 1.0, 1.0, 0.9, 1.1, 0.7, 0.8, 1.0, 1.0, 1.0, 1.0, -1.0, 1e-3, 50.0, 1.0])
    k = ints([3, 3, 4, 20, 0, 60, 100, 5, 5, 5, 10, 3, 5, 40, V, V + 5], "cpu")
    p = torch.tensor([0.9, 0.5, 1.0, 0.5, 0.99, 0.95, 0.9, 0.9, 0.9, 0.9, 0.9, 0.9, 0.5, 0.9, 0.3, 1.0])
    check_probabilities(logits, T, k, p)
    check_probabilities(logits, T, None, None)
    check_probabilities(logits, None, None, None)
    check_probabilities(logits[:1].repeat(300, 1)[:, :77].contiguous(), torch.full((300,), 0.6), ints([9] * 300, "cpu"), None)


@gpu
@pytest.mark.parametrize("V", [2500, 40001, 151936])
def test_probabilities_that_no_few_candidates_decide(V):
    """Rows so flat, a k so large or a mass so near its whole that the kept values' edge lies among thousands; rows with two values
    only; the same answer every time."""
    g = torch.Generator().manual_seed(V)
    logits = torch.randn(6, V, generator=g)
    logits[0] *= 1e-3
    logits[1] = 0.0
    logits[2] = (torch.rand(V, generator=g) < 0.5).float()
    logits[3, V // 2:] -= 60.0
    T, k, p = torch.full((6,), 1.0), ints([0, 0, 0, 0, V - 1, V // 2], "cpu"), [0.5, 0.3, 0.6, 0.9999, 1.0, 0.8]

    def halfway(T, k):
        """The masses as they are, but between those of two tokens: there the target is half a token's mass from either, more than
        the rounding of all terms by 2^-24 makes (two of the whole, 151,936 tokens: 0.02 of a token's mass where all are alike)."""
        made = []
        for r in range(6):
            x = (logits[r] * (torch.tensor(1.0) / T)).double().sort(descending=True).values[:k[r] or V]
            upto = torch.cumsum(torch.exp(x - x[0]), 0)
            at = int((upto >= p[r] * upto[-1]).nonzero()[0])
            made.append(float((upto[at] + upto[at - 1]) / 2 / upto[-1]) if p[r] < 1 else 1.0)
        return torch.tensor(made)

    check_probabilities(logits, 20 * T, None, halfway(20.0, [0] * 6))
    p = halfway(1.0, k.tolist())
    check_probabilities(logits, T, k, p)
    args = logits.to(DEV), T.to(DEV), k.to(DEV), p.to(DEV)
    first, again = torch.empty(6, V, device=DEV), torch.empty(6, V, device=DEV)
    ops.probabilities(args[0], first, *args[1:])
    for _ in range(5):
        ops.probabilities(args[0], again, *args[1:])
        assert torch.equal(first, again)


@gpu
@pytest.mark.parametrize("V", [5, 1027, 30002])
def test_probabilities_of_rows_that_begin_anywhere(V):
    g = torch.Generator().manual_seed(V)
    rows, T = 3 * torch.randn(4, V, generator=g), torch.tensor([0.7, 0.0, 1.2, 0.9])
    k, p = ints([0, 3, 20, 0], "cpu"), torch.tensor([0.8, 1.0, 0.9, 1.0])
    want = plain_probabilities(rows, T, k, p)
    for a, b in ((1, 0), (0, 3), (2, 2), (3, 1)):
        logits, out = torch.full((4 * V + 8,), 50.0, device=DEV), torch.full((4 * V + 8,), 7.0, device=DEV)
        logits[a:a + 4 * V] = rows.view(-1).to(DEV)
        ops.probabilities(logits[a:a + 4 * V].view(4, V), out[b:b + 4 * V].view(4, V), T.to(DEV), k.to(DEV), p.to(DEV))
        got = out[b:b + 4 * V].view(4, V).cpu().double()
        assert ((got > 0) == (want > 0)).all() and ((got - want).abs() <= 2.8e-6 * want).all()
        assert (out[:b] == 7.0).all() and (out[b + 4 * V:] == 7.0).all()


@gpu
@pytest.mark.parametrize("T,k,p", [(0.8, 50, 0.9), (1.0, 0, 0.8), (1.0, 8, 1.0)])
def test_probabilities_are_what_sample_draws_from(T, k, p):
    """Every drawn token has mass, and over many draws a token comes as often as its probability says."""
    g = torch.Generator().manual_seed(8)
    V, M = 300, 4096
    logits = (2.5 * torch.randn(1, V, generator=g)).repeat(M, 1).to(DEV)
    T, k, p = (torch.full((M,), x, dtype=d, device=DEV) for x, d in ((T, F32), (k, torch.int32), (p, F32)))
    out, drawn = torch.empty_like(logits), torch.empty(M, dtype=torch.int32, device=DEV)
    ops.probabilities(logits, out, T, k, p)
    ops.sample(logits, drawn, T, k, p, torch.arange(M, dtype=torch.int64, device=DEV), torch.zeros(M, dtype=torch.int32, device=DEV))
    assert (out == out[0]).all()
    w = out[0].double().cpu()
    often = torch.bincount(drawn.long().cpu(), minlength=V).double()
    assert (w[often > 0] > 0).all()
    assert ((often - M * w).abs() <= 5 * (M * w * (1 - w)).sqrt() + 1).all()


@gpu
@pytest.mark.parametrize("V,k", [(3000, 0), (3000, 500), (900, 0), (900, 300), (70001, 0)])
def test_probabilities_keep_what_sample_keeps(V, k):
    """Rows whose top-p lies, to 1e-10, where the mass of the largest tokens ends: whether the next one is kept hangs on how the
    masses are rounded, so both have to take the same ones.  That token has a sixth of the kept mass: of 128 draws none has it, where
    it is kept, once in 1e10."""
    g = torch.Generator().manual_seed(V + k)
    rows, draws = 24, 128
    logits, p = torch.empty(rows, V), torch.empty(rows)
    for r in range(rows):
        x = -5.0 - math.log(V / 900) - 3.0 * torch.rand(V, generator=g)
        large = torch.tensor([1.0, 0.8, 0.6, 0.5]) * (1 + 0.05 * torch.rand(4, generator=g))
        x[[5, 200, 310, 777]] = large.sort(descending=True).values.log()
        kept = x.sort(descending=True).indices[:k or V]
        w = torch.exp(x.double())
        before, total = w[[5, 200, 310]].sum(), w[kept].sum()
        p[r] = before / total                       # a float: the mass of one small token is moved to where it is right
        at = int(kept[20])
        x[at] = torch.log(w[at] + before / p[r].double() - total).float()
        logits[r] = x
    many = logits.repeat_interleave(draws, 0).to(DEV)
    M = rows * draws
    T, ks, ps = torch.ones(M, device=DEV), ints([k] * M), p.repeat_interleave(draws).to(DEV)
    out, drawn = torch.empty(rows, V, device=DEV), torch.empty(M, dtype=torch.int32, device=DEV)
    ops.sample(many, drawn, T, ks, ps, torch.arange(M, dtype=torch.int64, device=DEV), torch.zeros(M, dtype=torch.int32, device=DEV))
    ops.probabilities(logits.to(DEV), out, T[:rows].clone(), ks[:rows].clone(), p.to(DEV))
    sampled = (drawn.view(rows, draws) == 777).any(1).cpu()
    assert torch.isin(drawn, ints([5, 200, 310, 777])).all()
    assert torch.equal((out[:, 777] > 0).cpu(), sampled)
    assert (out > 0).sum(1).tolist() == [4 if s else 3 for s in sampled.tolist()]


@gpu
def test_probabilities_of_many_rows_of_a_large_vocabulary():
    """One block to a row, so that the histogram of a top-p alone has its fewest places, with masses that are all rounded the same
    way among the rows; a k beyond what the groups of so few blocks are good for, and one within."""
    g = torch.Generator().manual_seed(12)
    V, M = 152064, 520
    logits = 2.5 * torch.randn(4, V, generator=g)
    logits[1] = (logits[1] * 100).round() / 100         # few different ones, hundreds of each
    T, k, p = torch.tensor([0.9, 1.0, 1.1, 1.0]), ints([0, 0, 50, 20], "cpu"), torch.tensor([0.9, 0.7, 0.95, 1.0])
    want = plain_probabilities(logits, T, k, p)
    rows = torch.arange(M) % 4
    many, out = logits.to(DEV)[rows.to(DEV)].contiguous(), torch.empty(M, V, device=DEV)
    ops.probabilities(many, out, T[rows].to(DEV), k[rows].to(DEV), p[rows].to(DEV))
    got = out[:4].cpu().double()
    tiny = want < 1e-30
    assert ((got > 0) == (want > 0))[~tiny].all() and ((got - want).abs() <= 2.8e-6 * want)[~tiny].all()
    assert torch.equal(out, out[:4][rows.to(DEV)])


# ------------------------------------------------------------------------------------------------ verification
def plain_verify(p, q, tokens, parents, starts, u, depth):
    """Request by request, the residual kept whole and normalised after every refusal (float64)."""
    paths, drawn = [], []
    V = p.shape[1]
    for r in range(len(starts) - 1):
        base, n = starts[r], starts[r + 1] - starts[r]
        if n == 0:
            paths.append([])
            drawn.append(-1)
            continue
        path, here = [0], 0
        while True:
            whole = p[base + here].double()
            left, taken = whole, None
            for i in range(here + 1, n) if len(path) < depth else ():
                x = int(tokens[base + i])
                if int(parents[base + i]) != here or not 0 <= x < V:
                    continue
                draft = q[base + here].double() if q is not None else torch.zeros(V, dtype=torch.float64).index_fill_(0, torch.tensor([x]), 1.0)
                if float(u[base + i]) * float(draft[x]) < float(left[x]):
                    taken = i
                    break
                left = (left - draft).clamp(min=0)
                left = left / left.sum() if left.sum() > 0 else left
            if taken is None:
                break
            here = taken
            path.append(here)
        left = left if left.sum() > 0 else whole
        upto = torch.cumsum(left, 0)
        at = (upto > float(u[base]) * upto[-1]).nonzero()
        paths.append(path)
        drawn.append(int(at[0]) if at.numel() else 0)
    return paths, drawn


def make_drafts(trees, V, seed, with_q=True, near=0.7, width=3, sharp=1.0):
    g = torch.Generator().manual_seed(seed)
    rng = random.Random(seed)
    N = sum(trees)
    logits = sharp * 2 * torch.randn(N, V, generator=g)
    p, q = torch.softmax(logits, 1), torch.softmax(logits + near * torch.randn(N, V, generator=g), 1)
    starts, parents, tokens = [0], [], []
    for n in trees:
        tree = random_tree(rng, n, width)[:n]
        parents += tree
        for t in tree:
            tokens.append(int(torch.multinomial(q[starts[-1] + max(t, 0)], 1, generator=g)))
        starts.append(starts[-1] + n)
    return p, q if with_q else None, tokens, parents, starts, torch.rand(N, generator=g)


def run_verify(p, q, tokens, parents, starts, u, depth):
    R = len(starts) - 1
    nodes, counts, out = ints([[7] * depth] * R), ints([7] * R), ints([7] * R)
    ops.verify_drafts(p.to(DEV), None if q is None else q.to(DEV), ints(tokens), ints(parents), ints(starts), u.to(DEV), nodes, counts, out)
    return nodes.tolist(), counts.tolist(), out.tolist()


def check_verify(p, q, tokens, parents, starts, u, depth):
    paths, drawn = plain_verify(p, q, tokens, parents, starts, u, depth)
    nodes, counts, out = run_verify(p, q, tokens, parents, starts, u, depth)
    assert counts == [len(x) for x in paths]
    assert nodes == [x + [-1] * (depth - len(x)) for x in paths]
    assert out == drawn
    return paths, out


@gpu
@pytest.mark.parametrize("with_q", [True, False])
@pytest.mark.parametrize("V", [1, 2, 33, 1000, 1025, 20001])
@pytest.mark.parametrize("trees", [[1], [5], [1, 2, 0, 9, 3], [70]])
def test_verify_drafts(V, trees, with_q):
    lengths = set()
    for seed in range(6):
        paths, _ = check_verify(*make_drafts(trees, V, seed, with_q), max(trees))
        lengths |= {len(x) for x in paths}
    assert V == 1 or max(trees) < 5 or len(lengths) > 1 or not with_q      # (of the plain paths: the inputs reach several ends)


@gpu
def test_verify_drafts_of_a_large_vocabulary():
    for seed, with_q in ((1, True), (2, False), (3, True)):
        check_verify(*make_drafts([9, 1, 6], 152064, seed, with_q, near=1.0, sharp=1.5), 9)


@gpu
def test_verify_drafts_without_the_other_blocks():
    """A leader that does not wait for the other blocks of its request works every sum out itself, to the same result; so does one
    that waits hardly at all, whatever has come by then."""
    made = [make_drafts([9, 1, 6, 0, 30], 20001, seed, with_q, near=1.0) for seed, with_q in ((1, True), (2, False), (3, True))]
    want = [run_verify(*m, 30) for m in made]
    try:
        for looks in (-1, 1, 2):
            ops._get("ms_verify_drafts_patience")(looks)
            assert [run_verify(*m, 30) for m in made] == want
    finally:
        ops._get("ms_verify_drafts_patience")(0)
    for m in made:
        check_verify(*m, 30)


@gpu
def test_verify_drafts_of_long_trees_and_many_requests():
    """More tokens than a block keeps at hand, more children of one token than that, more requests than CUs."""
    p, q, tokens, parents, starts, u = make_drafts([1500, 3], 40, 3, True, near=1.5, width=2)
    check_verify(p, q, tokens, parents, starts, u, 64)
    check_verify(p, None, tokens, parents, starts, u, 64)
    parents[:1500] = [-1] + [0] * 1499
    u[:1500] = 1.0 - 2.0 ** -24
    p[0] = 0.0
    p[0, 39] = 1e-3
    p[0, 38] = 1.0 - 1e-3
    tokens[:1500] = [i % 38 for i in range(1500)]
    check_verify(p, None, tokens, parents, starts, u, 3)
    for with_q in (True, False):
        check_verify(*make_drafts([1 + i % 4 for i in range(400)], 1100, 6, with_q), 4)


@gpu
@pytest.mark.parametrize("with_q", [True, False])
def test_verify_drafts_edges(with_q):
    """Numbers of zero and next to one, equal distributions, guesses without mass, the same guess twice, guesses that are no
    tokens, paths that fill their place, distributions with one token."""
    p, q, tokens, parents, starts, u = make_drafts([6, 6, 6, 6, 6, 6], 50, 5, True)
    parents[12:18] = [-1, 0, 0, 0, 0, 0]
    tokens[12:18] = [0, 9, 9, 9, 9, 9]                   # the same guess again and again
    p[12, 9] = 0.0
    parents[18:24] = [-1, 0, 1, 2, 3, 4]
    u[18:24] = 0.0                                       # everything with mass is accepted, the first token with any drawn
    u[24:30] = 1.0 - 2.0 ** -24
    tokens[25], tokens[26] = -1, 50
    p[30] = torch.zeros(50)
    p[30, 17] = 1.0
    q[30] = p[30]
    tokens[30:36] = [3, 17, 17, 4, 17, 2]
    parents[30:36] = [-1, 0, 1, 0, 0, 2]
    q[0] = p[0]
    q = q if with_q else None
    for depth in (1, 2, 4, 6):
        check_verify(p, q, tokens, parents, starts, u, depth)
    # nothing left of the target: its own distribution; no distribution at all: token 0
    check_verify(torch.zeros(2, 9), None, [1, 2], [-1, 0], [0, 2], torch.tensor([0.5, 0.5]), 2)
    one = torch.full((1, 9), 1 / 9)
    check_verify(one, one, [4], [-1], [0, 1], torch.tensor([0.999]), 1)


@gpu
@pytest.mark.parametrize("with_q", [True, False])
def test_tokens_come_as_often_as_the_target_has_them(with_q):
    """Three guesses behind the root, drawn from q (or fixed), over many requests: the first token that comes out, accepted or
    drawn, is distributed as p."""
    g = torch.Generator().manual_seed(11)
    V, R = 6, 20000
    p = torch.tensor([0.30, 0.05, 0.22, 0.03, 0.25, 0.15])
    q = torch.tensor([0.10, 0.40, 0.20, 0.20, 0.05, 0.05])
    guesses = torch.multinomial(q.repeat(R, 1), 3, replacement=True, generator=g) if with_q else torch.tensor([[1, 0, 1]]).repeat(R, 1)
    tokens = torch.cat([torch.zeros(R, 1, dtype=torch.long), guesses], 1).flatten().tolist()
    rows = p.repeat(4 * R, 1)
    nodes, counts, out = run_verify(rows, q.repeat(4 * R, 1) if with_q else None, tokens, [-1, 0, 0, 0] * R, list(range(0, 4 * R + 1, 4)),
                                    torch.rand(4 * R, generator=g), 4)
    first = [tokens[4 * r + nodes[r][1]] if counts[r] > 1 else out[r] for r in range(R)]
    often = torch.bincount(torch.tensor(first), minlength=V).double()
    assert ((often - R * p).abs() <= 5 * (R * p * (1 - p)).sqrt()).all(), often / R
    assert 0.2 * R < sum(c > 1 for c in counts) < R


# ------------------------------------------------------------------------------------------------ the cache
def make_pages(dtype, L, heads, width, page_size, contexts, transposed, seed=0):
    g = torch.Generator().manual_seed(seed)
    rng = random.Random(seed)
    need = [-(-c // page_size) for c in contexts]
    order = list(range(1, sum(need) + 1))
    rng.shuffle(order)
    rows = list(range(len(contexts) + 1))
    rng.shuffle(rows)
    table = torch.zeros(len(contexts) + 1, max(need) + 1, dtype=torch.int32)
    for r, n in enumerate(need):
        for b in range(n):
            table[rows[r], b] = order.pop()
    shape = (width, page_size) if transposed else (page_size, width)
    return torch.randn(L, sum(need) + 1, heads, *shape, generator=g).to(dtype), table, rows[:len(contexts)]


def plain_keep(pages, transposed, table, rows, first, nodes, counts):
    out = pages.clone()
    size = pages.shape[4] if transposed else pages.shape[3]
    for r, path in enumerate(nodes):
        for i, n in enumerate(path[:counts[r]]):
            a, b = first[r] + n, first[r] + i
            if a // size >= table.shape[1]:
                continue
            pa, pb = int(table[rows[r], a // size]), int(table[rows[r], b // size])
            if not (0 < pa < pages.shape[1] and 0 < pb < pages.shape[1]):
                continue
            if transposed:
                out[:, pb, :, :, b % size] = pages[:, pa, :, :, a % size]
            else:
                out[:, pb, :, b % size] = pages[:, pa, :, a % size]
    return out


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("L,heads,width,page_size", [(3, 2, 64, 16), (1, 1, 20, 7), (2, 3, 33, 16), (5, 2, 128, 32), (2, 8, 128, 1)])
def test_keep_tokens(dtype, L, heads, width, page_size):
    contexts, trees = [9, 40, 100, 64, 33], [9, 20, 70, 5, 32]
    paths = [[0, 3, 4, 8], [0], [0, 1, 2, 3, 17, 18, 40, 69], [], [0, 1, 31]]
    depth = 9
    counts = [len(x) for x in paths]
    nodes = [x + [-1] * (depth - len(x)) for x in paths]
    first = [c - t for c, t in zip(contexts, trees)]
    made = [make_pages(dtype, L, h, w, page_size, contexts, flip) for h, w, flip in ((heads, width, False), (heads, width, True), (1, 16, True))]
    table, rows = made[0][1:]
    pages = [m[0].to(DEV) for m in made]
    flips = [False, True, True]
    ops.keep_tokens(pages, flips, table.to(DEV), ints(first), ints(nodes), ints(counts), ints(rows))
    for got, m, flip in zip(pages, made, flips):
        assert torch.equal(got.cpu(), plain_keep(m[0], flip, table, rows, first, nodes, counts))
    # a single layer without its dimension, as a run's view has it, and the table's rows in order
    one = made[1][0][0].to(DEV).contiguous()
    ops.keep_tokens([one], [True], table[rows].to(DEV).contiguous(), ints(first), ints(nodes), ints(counts))
    assert torch.equal(one.cpu(), plain_keep(made[1][0][:1], True, table, rows, first, nodes, counts)[0])


@gpu
def test_keep_tokens_of_a_long_path_and_of_pages_given_back():
    """Longer paths than a block reads at once; entries on the null page, behind the table or on pages outside the pool stay."""
    path = [0] + list(range(3, 300, 2))
    pages, table, rows = make_pages(BF16, 2, 2, 64, 16, [400, 400], True)
    nodes, counts = [path, path], [len(path), 400]
    first = [100, 90]
    table[rows[1], 7] = 0
    table[rows[1], 9] = pages.shape[1] + 3
    table[rows[1], 12] = -5
    nodes[1] = path[:-1] + [10 ** 6]
    got = pages.to(DEV)
    ops.keep_tokens([got], [True], table.to(DEV), ints(first), ints(nodes), ints(counts), ints(rows))
    assert torch.equal(got.cpu(), plain_keep(pages, True, table, rows, first, nodes, counts))


# ------------------------------------------------------------------------------------------------ together
class Toy:
    """One layer of attention over embedded tokens and a head, enough for a target whose next token depends on all before it."""

    def __init__(self, dtype, nh=4, nkv=2, d=64, V=97, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.nh, self.nkv, self.d, self.V, self.dtype = nh, nkv, d, V, dtype
        self.qkv = (torch.randn(V, (nh + 2 * nkv) * d, generator=g)).to(dtype).to(DEV)
        self.place = torch.randn(512, nkv * d, generator=g).to(DEV)      # added to the keys by position
        self.head = (torch.randn(nh * d, V, generator=g) * 0.5).to(DEV)

    def project(self, tokens, positions):
        x = self.qkv[tokens.long()].clone()
        at = slice(self.nh * self.d, (self.nh + self.nkv) * self.d)
        x[:, at] = (x[:, at].float() + self.place[positions.long()]).to(self.dtype)
        return x

    def store(self, kv, x, req, slots, table):
        k = x[:, self.nh * self.d:(self.nh + self.nkv) * self.d].view(-1, self.nkv, self.d)
        v = x[:, (self.nh + self.nkv) * self.d:].view(-1, self.nkv, self.d)
        page, slot = table[req.long(), slots.long() // 16].long(), slots.long() % 16
        kv.k_pages[page, :, slot] = k
        if kv.v_transposed:
            kv.v_pages[page, :, :, slot] = v
        else:
            kv.v_pages[page, :, slot] = v

    def logits(self, out):
        return out.float() @ self.head


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("temperature", [0.0, 0.9])
def test_a_step_of_all_of_them(dtype, temperature):
    """Steps of trees over a cache: what they accept is what the distributions say, and a cache that such steps left holds the
    same entries, and answers the next step alike, as one that saw only the accepted tokens."""
    toy, rng, g = Toy(dtype), random.Random(2), torch.Generator().manual_seed(3)
    R, pages = 3, 12
    flip = dtype == BF16
    table = (torch.arange(R * pages, dtype=torch.int32).view(R, pages) + 1).to(DEV)

    def empty():
        shape = (R * pages + 1, toy.nkv, 16, toy.d)
        return SimpleNamespace(k_pages=torch.zeros(shape, dtype=dtype, device=DEV), v_transposed=flip, block_table=table, table_rows=None,
                               v_pages=torch.zeros((shape[0], toy.nkv, toy.d, 16) if flip else shape, dtype=dtype, device=DEV))

    kv = empty()
    known = [[rng.randrange(toy.V) for _ in range(n)] for n in (5, 30, 17)]     # the last token of each is not in the cache yet
    for r in range(R):
        n = len(known[r]) - 1
        pos = ints(list(range(n)))
        toy.store(kv, toy.project(ints(known[r][:-1]), pos), ints([r] * n), pos, table)
    lengths = set()
    for step in range(6):
        trees = [rng.randint(3, 12) for _ in range(R)]
        parents = [random_tree(rng, n) for n in trees]
        starts = [0, trees[0], trees[0] + trees[1], sum(trees)]
        N, flat = sum(trees), sum(parents, [])
        before = [len(x) - 1 for x in known]
        owner = [r for r, n in enumerate(trees) for _ in range(n)]
        depth, tokens = [], []
        for n, (r, up) in enumerate(zip(owner, flat)):
            depth.append(0 if up < 0 else depth[starts[r] + up] + 1)
            tokens.append(known[r][-1] if up < 0 else rng.randrange(toy.V))
        likes = [rng.random() < 0.7 for _ in range(N)]
        positions, places = ints([before[r] + d for r, d in zip(owner, depth)]), ints([before[r] + n - starts[r] for n, r in enumerate(owner)])
        ctx = SimpleNamespace(token_req=ints(owner), q_start=ints(starts), context_lens=ints([b + n for b, n in zip(before, trees)]),
                              max_q_len=max(trees), max_context_len=max(b + n for b, n in zip(before, trees)), n_live_tokens=None)
        tree = ints([w for t in parents for w in mask_words(ancestors(t), 1)])
        out, p = torch.empty(N, toy.nh * toy.d, dtype=dtype, device=DEV), torch.empty(N, toy.V, device=DEV)
        # level by level, so that some guesses are what the target likes best behind their parent
        for level in range(max(depth) + 1):
            x = toy.project(ints(tokens), positions)
            toy.store(kv, x, ctx.token_req, places, table)
            ops.tree_attention(x[:, :toy.nh * toy.d], kv, ctx, tree, out, toy.nh, 0.1)
            ops.probabilities(toy.logits(out), p, torch.full((N,), temperature, device=DEV), ints([40] * N), torch.full((N,), 0.95, device=DEV))
            best = p.argmax(dim=1).tolist()
            for n in range(N):
                if depth[n] == level + 1 and likes[n]:
                    tokens[n] = best[starts[owner[n]] + flat[n]]
        u = torch.rand(N, generator=g)
        nodes, counts, drawn = ints([[7] * 12] * R), ints([0] * R), ints([0] * R)
        ops.verify_drafts(p, None, ints(tokens), ints(flat), ints(starts), u.to(DEV), nodes, counts, drawn)
        paths, want = plain_verify(p.cpu(), None, tokens, flat, starts, u, 12)
        assert drawn.tolist() == want and [c[:n] for c, n in zip(nodes.tolist(), counts.tolist())] == paths
        lengths |= set(counts.tolist())
        ops.keep_tokens([kv.k_pages, kv.v_pages], [False, flip], table, ints(before), nodes, counts)
        for r in range(R):
            known[r] = known[r] + [tokens[starts[r] + n] for n in paths[r][1:]] + [want[r]]
    assert len(lengths) > 1
    fresh = empty()
    for r in range(R):
        n = len(known[r]) - 1
        pos = ints(list(range(n)))
        toy.store(fresh, toy.project(ints(known[r][:-1]), pos), ints([r] * n), pos, table)
        at = torch.arange(n, device=DEV)
        page, slot = table[r, at // 16].long(), at % 16
        assert torch.equal(kv.k_pages[page, :, slot], fresh.k_pages[page, :, slot])
        pick = (lambda c: c.v_pages[page, :, :, slot]) if flip else (lambda c: c.v_pages[page, :, slot])
        assert torch.equal(pick(kv), pick(fresh))
    # a decode step goes on behind them
    last, lens = ints([x[-1] for x in known]), [len(x) for x in known]
    results = []
    for cache in (kv, fresh):
        x = toy.project(last, ints(lens) - 1)
        toy.store(cache, x, ints([0, 1, 2]), ints(lens) - 1, table)
        out = torch.empty(R, toy.nh * toy.d, dtype=dtype, device=DEV)
        ops.paged_attention_generic(x[:, :toy.nh * toy.d], cache.k_pages, cache.v_pages, table, ints([0, 1, 2]), ints(lens) - 1, out, toy.nh, 0.1,
                                    v_transposed=flip)
        results.append(out)
    assert torch.equal(*results)


@gpu
def test_the_step_replays_from_a_graph():
    """Captured on a stream of its own and replayed over changed inputs, with eager work between; every replay against the eager
    call."""
    s = make_step(BF16, 14, 2, 64, 16, [8, 5, 13], [300, 40, 2000], seed=1)
    N, V = 26, 5003
    drafts = [make_drafts([8, 5, 13], V, seed) for seed in range(4)]
    p, q, tokens, parents, starts, u = [x.to(DEV) if torch.is_tensor(x) else ints(x) for x in drafts[0]]
    logits, T = torch.empty(N, V, device=DEV), torch.full((N,), 0.8, device=DEV)
    k, pr = ints([40] * N), torch.full((N,), 0.9, device=DEV)
    made, probs = torch.empty_like(logits), torch.empty_like(logits)
    nodes, counts, drawn = ints([[0] * 13] * 3), ints([0] * 3), ints([0] * 3)
    first = s.ctx.context_lens - ints([8, 5, 13])

    def step():
        ops.tree_attention(s.q, s.kv, s.ctx, s.tree, s.out, 14, s.scale)
        ops.probabilities(logits, made, T, k, pr)
        ops.probabilities(logits, probs, T)
        ops.verify_drafts(p, q, tokens, parents, starts, u, nodes, counts, drawn)
        ops.keep_tokens([s.kv.k_pages, s.kv.v_pages], [False, True], s.kv.block_table, first, nodes, counts, s.kv.table_rows)

    side = torch.cuda.Stream()
    cached = s.kv.k_pages.clone(), s.kv.v_pages.clone()
    logits.normal_()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.inference_mode(), torch.cuda.graph(graph, stream=side):     # (as the engine captures: the generator keeps the first mode)
        step()
    results = []
    for i in range(1, 4):
        for to, of in zip((p, q, tokens, parents, starts, u), drafts[i]):
            to.copy_(of.to(DEV) if torch.is_tensor(of) else ints(of))
        logits.normal_(generator=torch.Generator(device=DEV).manual_seed(i))
        s.q.normal_(generator=torch.Generator(device=DEV).manual_seed(i))
        both = []
        for run in (graph.replay, step):
            s.kv.k_pages.copy_(cached[0])
            s.kv.v_pages.copy_(cached[1])
            for t in (s.out, made, probs):
                t.fill_(5.0)
            for t in (nodes, counts, drawn):
                t.fill_(5)
            run()
            torch.cuda.synchronize()
            both.append([t.clone() for t in (s.out, made, probs, nodes, counts, drawn, s.kv.k_pages, s.kv.v_pages)])
        for a, b in zip(*both):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
        results.append(both[0][3].tolist())
    assert results[0] != results[1] or results[1] != results[2]


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_calls_without_requests_or_tokens(dtype):
    """No requests: tokens that pad the batch stay; requests without tokens: empty paths, no token, nothing moved."""
    for d in (64, 48):
        s = make_step(dtype, 4, 2, d, 16, [3], [20])
        s.ctx.q_start, s.ctx.context_lens, s.kv.table_rows = ints([0]), ints([]), ints([])
        ops.tree_attention(s.q, s.kv, s.ctx, s.tree, s.out, 4, s.scale)
        assert (s.out == 7.0).all()
        s = make_step(dtype, 4, 2, d, 16, [0, 0], [20, 0])
        assert ops.tree_attention(s.q, s.kv, s.ctx, s.tree, s.out, 4, s.scale).shape == (0, 4 * d)
    assert ops.probabilities(torch.empty(0, 50, device=DEV), torch.empty(0, 50, device=DEV)).shape == (0, 50)
    for with_q in (True, False):
        q = torch.empty(0, 50) if with_q else None
        nodes, counts, out = run_verify(torch.empty(0, 50), q, [], [], [0, 0, 0], torch.empty(0), 3)
        assert nodes == [[-1] * 3] * 2 and counts == [0, 0] and out == [-1, -1]
    none = ints([])
    ops.verify_drafts(torch.empty(0, 50, device=DEV), None, none, none, ints([0]), torch.empty(0, device=DEV), none.view(0, 3), none, none)
    pages, table, _ = make_pages(dtype, 2, 2, 64, 16, [40, 20], False)
    got = pages.to(DEV)
    ops.keep_tokens([got], [False], table.to(DEV), ints([30, 15]), ints(nodes), ints(counts))
    assert torch.equal(got.cpu(), pages)


@gpu
def test_calls_on_two_streams_at_once():
    """Each has its own workspace, and a verification whose blocks wait for each other shares the chip with another's."""
    made = [make_drafts([9, 1, 6, 0, 30] * 8, 20001, seed, True, near=1.0) for seed in (1, 2)]
    on = [[x.to(DEV) if torch.is_tensor(x) else ints(x) for x in m] for m in made]
    steps = [make_step(BF16, 14, 2, 64, 16, [8, 5, 13], [300, 40, 2000], seed=seed) for seed in (1, 2)]
    R, N = 40, on[0][0].shape[0]
    T, pr = torch.full((N,), 0.8, device=DEV), torch.full((N,), 0.9, device=DEV)

    def run(i):
        p, q, tokens, parents, starts, u = on[i]
        nodes, counts, out = ints([[7] * 30] * R), ints([7] * R), ints([7] * R)
        made, s = torch.empty_like(p), steps[i]
        ops.probabilities(p, made, T, None, pr)
        ops.verify_drafts(p, q, tokens, parents, starts, u, nodes, counts, out)
        ops.tree_attention(s.q, s.kv, s.ctx, s.tree, s.out, 14, s.scale)
        return made, nodes, counts, out, s.out.clone()

    want = [run(i) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(4):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(run(i))
    torch.cuda.synchronize()
    for i in range(2):
        for results in got[i]:
            for a, b in zip(want[i], results):
                assert torch.equal(a, b)
    paths, drawn = plain_verify(*made[0], 30)
    assert want[0][2].tolist() == [len(x) for x in paths] and want[0][3].tolist() == drawn


@gpu
def test_the_sampler_and_the_pools_reach_them():
    """``Sampler.probabilities`` and ``verify`` against the operators with the same settings; ``CachePools.keep_tokens`` moves the
    entries of every group."""
    from llm_infrence_engine_amd.cache.manager import CacheLayout
    from llm_infrence_engine_amd.cache.pools import CachePools
    from llm_infrence_engine_amd.parts.base import CacheNeed, PageTensor, Runtime
    from llm_infrence_engine_amd.sampling.sampler import Sampler

    g = torch.Generator().manual_seed(5)
    rows = [SimpleNamespace(temperature=t, top_k=k, top_p=p) for t, k, p in ((0.8, 20, 0.9), (0.0, 5, 0.5), (1.2, 0, 1.0), (0.7, 0, 0.8))]
    logits = 2 * torch.randn(4, 700, generator=g)
    sampler = Sampler(torch.device(DEV))
    got = sampler.probabilities(logits.to(DEV), rows).cpu().double()
    want = plain_probabilities(logits, torch.tensor([r.temperature for r in rows]), ints([r.top_k for r in rows], "cpu"), torch.tensor([r.top_p for r in rows]))
    assert ((got - want).abs() <= 2.8e-6 * want + 1e-30).all()
    greedy = [SimpleNamespace(temperature=0.0, top_k=0, top_p=1.0)] * 4
    assert torch.equal(sampler.probabilities(logits.to(DEV), greedy).argmax(1).cpu(), logits.argmax(1))
    with pytest.raises(ValueError):
        sampler.probabilities(logits.to(DEV), rows[:3])
    made = make_drafts([5, 9], 300, 2)
    paths, drawn = plain_verify(*made, 9)
    p, q, tokens, parents, starts, u = made
    nodes, counts, out = sampler.verify(p.to(DEV), q.to(DEV), ints(tokens), ints(parents), ints(starts), u.to(DEV), 9)
    assert counts.tolist() == [len(x) for x in paths] and out.tolist() == drawn and [n[:c] for n, c in zip(nodes.tolist(), counts.tolist())] == paths

    rt = Runtime(device=torch.device(DEV), dtype=BF16)
    wide = CacheNeed((PageTensor("k", 2, 64), PageTensor("v", 2, 64, transpose_at=16)), None)
    narrow = CacheNeed((PageTensor("k", 1, 32), PageTensor("v", 1, 32, transpose_at=16)), 40)
    pools = CachePools(CacheLayout([(wide, None, None), (narrow, None, None), (wide, None, None)]), 16, 8, 2, rt, 4)
    for table, row in zip(pools.tables, ([3, 1, 2, 0], [5, 0, 7, 4])):
        table[1] = ints(row)
    before = []
    for pages in pools.pages:
        for t in pages.values():
            t.normal_(generator=torch.Generator(device=DEV).manual_seed(1))
        before.append({n: t.cpu().clone() for n, t in pages.items()})
    pools.keep_tokens(ints([30]), ints([[0, 2, 5, -1]]), ints([3]), ints([1]))
    for pages, flips, table, old in zip(pools.pages, pools.transposed, pools.tables, before):
        assert flips["v"] and not flips["k"]
        for n, t in pages.items():
            assert torch.equal(t.cpu(), plain_keep(old[n], flips[n], table.cpu(), [1], [30], [[0, 2, 5]], [3]))


# ------------------------------------------------------------------------------------------------ refusals (no GPU needed)
@pytest.fixture
def host(monkeypatch):
    """The checks on host tensors: they are told that everything is on the GPU, and what would be launched is noted."""
    monkeypatch.setattr(torch.Tensor, "is_cuda", True, raising=False)
    launched = []
    monkeypatch.setattr(ops, "_here", lambda *a: None)
    monkeypatch.setattr(ops, "_device", lambda: -1)
    monkeypatch.setattr(ops, "_call", lambda name, *a: launched.append(name))
    monkeypatch.setattr(ops, "_stream", lambda: 0)
    monkeypatch.setattr(ops, "_get", lambda name: (lambda *a: 64))      # (sizes of workspaces)
    return launched


def refused(launched, call, error=(ValueError, TypeError)):
    with pytest.raises(error):
        call()
    assert not launched


def test_ops_of_trees_run_on_the_gpu_only():
    z = torch.zeros(2, 5)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError):
        ops.probabilities(z, torch.zeros(2, 5))
    with pytest.raises(RuntimeError):
        ops.verify_drafts(z, None, i, i, i, z[:, 0], i.view(1, 2), i[:1], i[:1])
    with pytest.raises(RuntimeError):
        ops.keep_tokens([torch.zeros(2, 2, 2, 2)], [False], i.view(1, 2), i[:1], i.view(1, 2), i[:1])


@gpu
def test_the_library_takes_as_many_tensors_as_the_module_says():
    assert ops._get("ms_keep_tokens_max")() == ops.MAX_KEPT_TENSORS


def test_probabilities_refuse(host):
    z, out = torch.zeros(3, 8), torch.zeros(3, 8)
    T = torch.ones(3)
    refused(host, lambda: ops.probabilities(z, z, T))
    refused(host, lambda: ops.probabilities(z[:2], torch.zeros(3, 8), T[:2]))
    refused(host, lambda: ops.probabilities(z.double(), out, T))
    refused(host, lambda: ops.probabilities(z.t(), out.t(), T))
    refused(host, lambda: ops.probabilities(z, out, torch.ones(2)))
    refused(host, lambda: ops.probabilities(z, out, T, top_k=torch.ones(3)))
    refused(host, lambda: ops.probabilities(z, out, T, top_p=torch.ones(3, dtype=torch.float64)))
    refused(host, lambda: ops.probabilities(z[0], out[0], T))
    both = torch.zeros(4, 8)
    refused(host, lambda: ops.probabilities(both[:3], both[1:], T))
    ops.probabilities(z[:0], out[:0], T[:0])
    assert not host
    ops.probabilities(z, out, T)
    assert host == ["ms_probabilities"]


def test_verify_drafts_refuses(host):
    def args(**kw):
        i = lambda *v: torch.tensor(v, dtype=torch.int32)     # noqa: E731
        a = dict(p=torch.zeros(5, 9), q=torch.zeros(5, 9), token_ids=i(0, 1, 2, 3, 4), parents=i(-1, 0, 0, -1, 0), q_start=i(0, 3, 5),
                 uniforms=torch.zeros(5), nodes=torch.zeros(2, 3, dtype=torch.int32), counts=i(0, 0), out=i(0, 0))
        a.update(kw)
        return ops.verify_drafts(**a)

    i32 = torch.int32
    for kw in (dict(p=torch.zeros(5, 9).bfloat16()), dict(p=torch.zeros(5, 0)), dict(q=torch.zeros(5, 8)), dict(q=torch.zeros(4, 9)),
               dict(token_ids=torch.zeros(5, dtype=torch.int64)), dict(token_ids=torch.zeros(4, dtype=i32)), dict(parents=torch.zeros(6, dtype=i32)),
               dict(uniforms=torch.zeros(5).double()), dict(nodes=torch.zeros(3, 3, dtype=i32)), dict(nodes=torch.zeros(2, 0, dtype=i32)),
               dict(counts=torch.zeros(3, dtype=i32)), dict(out=torch.zeros(2)), dict(q_start=torch.zeros(0, dtype=i32)),
               dict(p=torch.zeros(9, 5).t())):
        refused(host, lambda: args(**kw))
    args()
    args(q=None)
    assert host == ["ms_verify_drafts"] * 2


def test_keep_tokens_refuses(host):
    def args(**kw):
        z = lambda *s: torch.zeros(*s, dtype=torch.int32)     # noqa: E731
        a = dict(pages=[torch.zeros(2, 7, 3, 16, 8), torch.zeros(2, 7, 3, 8, 16)], transposed=[False, True], block_table=z(4, 5), first=z(2),
                 nodes=z(2, 3), counts=z(2), table_rows=z(2))
        a.update(kw)
        return ops.keep_tokens(**a)

    i32 = torch.int32
    for kw in (dict(pages=[]), dict(transposed=[False]), dict(transposed=[True, True]), dict(pages=[torch.zeros(2, 7, 3, 16, 8), torch.zeros(2, 8, 3, 8, 16)]),
               dict(pages=[torch.zeros(2, 7, 3, 16, 8), torch.zeros(2, 7, 3, 8, 16).bfloat16()]), dict(pages=[torch.zeros(7, 3, 16)] * 2),
               dict(pages=[torch.zeros(2, 7, 3, 16, 8).half()] * 2, transposed=[False] * 2), dict(first=torch.zeros(3, dtype=i32)),
               dict(counts=torch.zeros(2, dtype=torch.int64)), dict(nodes=torch.zeros(2, dtype=i32)), dict(table_rows=torch.zeros(3, dtype=i32)),
               dict(table_rows=None, block_table=torch.zeros(1, 5, dtype=i32)), dict(pages=[torch.zeros(2, 7, 3, 16, 8)] * 17, transposed=[False] * 17),
               dict(pages=[torch.zeros(2, 7, 3, 16, 8)] * 2, transposed=[False] * 2)):
        refused(host, lambda: args(**kw))
    args(nodes=torch.zeros(2, 0, dtype=i32))
    assert not host
    args()
    assert host == ["ms_keep_tokens"]


def test_tree_attention_refuses(host):
    def args(q=None, out=None, tree=None, heads=4, flip=False, **kw):
        z = lambda *s: torch.zeros(*s, dtype=torch.int32)     # noqa: E731
        kv = SimpleNamespace(k_pages=torch.zeros(5, 2, 4, 24), v_pages=torch.zeros(5, 2, 4, 24), v_transposed=flip, block_table=z(3, 2), table_rows=z(2))
        ctx = SimpleNamespace(token_req=z(6), q_start=z(3), context_lens=z(2), max_q_len=4, max_context_len=8, n_live_tokens=None)
        for k, v in kw.items():
            setattr(kv if hasattr(kv, k) else ctx, k, v)
        return ops.tree_attention(torch.zeros(6, 96) if q is None else q, kv, ctx, z(6, 1) if tree is None else tree,
                                  torch.zeros(6, 96) if out is None else out, heads, 0.5)

    i32 = torch.int32
    refused(host, lambda: args(q=torch.zeros(6, 95)))
    refused(host, lambda: args(q=torch.zeros(96, 6).t()))
    refused(host, lambda: args(q=torch.zeros(6, 96).bfloat16()))
    refused(host, lambda: args(out=torch.zeros(6, 97)))
    refused(host, lambda: args(out=torch.zeros(5, 96)))
    refused(host, lambda: args(heads=3, out=torch.zeros(6, 72)))
    refused(host, lambda: args(tree=torch.zeros(6, 0, dtype=i32)))
    refused(host, lambda: args(tree=torch.zeros(5, 1, dtype=i32)))
    refused(host, lambda: args(tree=torch.zeros(6, 1, dtype=torch.int64)))
    refused(host, lambda: args(max_q_len=33))
    refused(host, lambda: args(flip=True))
    refused(host, lambda: args(v_pages=torch.zeros(4, 2, 4, 24)))
    refused(host, lambda: args(q_start=torch.zeros(2, dtype=i32)))
    refused(host, lambda: args(token_req=torch.zeros(5, dtype=i32)))
    refused(host, lambda: args(table_rows=torch.zeros(3, dtype=i32)))
    refused(host, lambda: args(table_rows=None, block_table=torch.zeros(1, 2, dtype=i32)))
    refused(host, lambda: args(context_lens=torch.zeros(2)))
    args()
    assert host == ["ms_tree_attention_generic"]
    wide = dict(q=torch.zeros(6, 128), out=torch.zeros(6, 128), k_pages=torch.zeros(5, 2, 4, 32), v_pages=torch.zeros(5, 2, 4, 32))
    del host[:]
    refused(host, lambda: args(max_context_len=9, **wide))
    refused(host, lambda: args(v_pages=torch.zeros(5, 2, 32, 4), **{k: v for k, v in wide.items() if k != "v_pages"}))
    refused(host, lambda: args(**{**wide, "out": torch.zeros(6, 128).bfloat16()}))
    args(**wide)
    assert host == ["ms_tree_attention_f32"]


def tree_call(width=24, N=6, R=2, **kw):
    """``tree_attention`` of host tensors: width 24 goes to the kernel for any size, 32 to the matrix cores; ``kw`` goes to the view where it
    has such a field, else to the context."""
    from llm_infrence_engine_amd.parts.base import KVView, StepContext

    z = lambda *s: torch.zeros(*s, dtype=torch.int32)     # noqa: E731
    pages = torch.zeros(5, 2, 4, width), torch.zeros(5, 2, 4, width)
    kv = KVView({"k": pages[0], "v": pages[1]}, {"k": False, "v": False}, z(3, 2), z(N), table_rows=z(R))
    ctx = StepContext(N, R, z(N), z(N), z(N), z(R + 1), z(R), z(R), z(N), 4, 8)
    for name, value in kw.items():
        setattr(kv if hasattr(kv, name) else ctx, name, value)
    return ops.tree_attention(torch.zeros(N, 4 * width), kv, ctx, z(N, 1), torch.zeros(N, 4 * width), 4, 0.5)


@pytest.mark.parametrize("width,kernel", [(24, "ms_tree_attention_generic"), (32, "ms_tree_attention_f32")])
def test_tree_attention_refuses_steps_without_bounds(host, width, kernel):
    """A step with tokens says how long its trees and contexts are at most (its context has 0 for both unless told)."""
    for kw in (dict(max_q_len=0), dict(max_context_len=0), dict(max_q_len=0, max_context_len=0), dict(max_context_len=3), dict(max_context_len=9)):
        refused(host, lambda: tree_call(width, **kw))
    assert tree_call(width, N=0, max_q_len=0, max_context_len=0).shape == (0, 4 * width)
    tree_call(width, R=0, max_q_len=0, max_context_len=0)
    assert not host
    tree_call(width)
    tree_call(width, max_context_len=4)
    assert host == [kernel] * 2


@pytest.mark.parametrize("width", [24, 32])
def test_tree_attention_refuses_views_with_a_window_or_entries_of_several_tokens(host, width):
    for kw in (dict(window=4), dict(window=4096), dict(stride=2)):
        refused(host, lambda: tree_call(width, **kw))
    tree_call(width, window=None, stride=1)
    assert len(host) == 1


def test_steps_that_the_matrix_kernel_has_no_room_for_go_to_the_other(host, monkeypatch):
    """Sizes that its plan, or its launch, does not take are the vector kernel's; what is wrong for either is refused."""
    monkeypatch.setattr(ops, "_get", lambda name: lambda *a: 0)
    tree_call(32)
    assert host == ["ms_tree_attention_generic"]
    monkeypatch.setattr(ops, "_get", lambda name: lambda *a: 64)
    call = ops._call

    def no_room(name, *a):
        if name == "ms_tree_attention_f32":
            raise ops.UnsupportedShape(name)
        call(name, *a)

    monkeypatch.setattr(ops, "_call", no_room)
    tree_call(32)
    assert host == ["ms_tree_attention_generic"] * 2
    del host[:]
    refused(host, lambda: tree_call(32, max_context_len=9))


def test_the_plan_of_the_longest_contexts_fits_its_number():
    """Up to its last bound of keys the plan names a kind there is and a share of them, for few blocks as for many."""
    for R, N, nh, nkv, d in ((1, 1, 14, 2, 64), (512, 512, 14, 2, 64), (65535, 65535, 32, 8, 128), (1024, 4096, 32, 1, 128)):
        for keys in (64, 64 * 65534, 64 * 65535):
            plan = ops._get("ms_tree_attention_mfma_plan")(R, N, 1 if N == R else 8, keys, nh, nkv, d, 16)
            share = (plan & 0xFFFF) * 64
            assert 0 <= plan >> 16 < 4 and share > 0 and -(-keys // share) <= 128
        assert ops._get("ms_tree_attention_mfma_plan")(R, N, 1, 64 * 65535 + 1, nh, nkv, d, 16) == -1


def test_keep_tokens_refuses_page_tensors_that_share_memory(host):
    z = lambda *s: torch.zeros(*s, dtype=torch.int32)     # noqa: E731
    call = lambda *pages: ops.keep_tokens(list(pages), [False] * len(pages), z(4, 5), z(2), z(2, 3), z(2), z(2))     # noqa: E731
    pool = torch.zeros(3, 7, 2, 16, 8)
    other = torch.zeros(2, 7, 2, 16, 8)
    refused(host, lambda: call(pool[:2], pool[1:]))
    refused(host, lambda: call(pool[1:], other, pool[:2]))
    refused(host, lambda: call(pool, pool))
    refused(host, lambda: call(other, other.view(-1).view(2, 7, 2, 16, 8)))
    call(pool[0], pool[1], pool[2])
    call(pool[:2], other)
    assert host == ["ms_keep_tokens"] * 2


def test_pools_that_cannot_drop_tokens_refuse(host):
    from llm_infrence_engine_amd.cache.pools import CachePools

    z = torch.zeros(1, dtype=torch.int32)
    for state, strides in (({0: ()}, [1]), ({}, [1, 4])):
        pools = CachePools.__new__(CachePools)
        pools.state, pools.layout = state, SimpleNamespace(group_keys=[SimpleNamespace(stride=s) for s in strides])
        refused(host, lambda: pools.keep_tokens(z, z.view(1, 1), z, z))
