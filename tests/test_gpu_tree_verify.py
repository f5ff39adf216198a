"""fg_tree_verify and fg_tree_accept against the definition in 64 bits: the
target's distribution after each rejection is formed whole, over the whole
vocabulary. Tokens, paths and counts must be equal: both sides work in 64 bits,
so they could differ only where a random number meets a border to 1e-15."""
import numpy as np
import pytest
import torch

from ferrolm_amd import gpu

pytestmark = pytest.mark.gpu


def positive(x):
    x = np.asarray(x, np.float64)
    return np.where(x > 0, x, 0.0)


def walk(parents, tokens, p, q, u, drafts):
    """(tokens, path) of one sequence by the definition."""
    out, path, node = [], [0], 0
    while True:
        target = positive(p[node])
        left, draft, total = target.copy(), None if q is None else positive(q[node]), 1.0
        drawn = 0.0  # without replacement: the mass of the tokens drawn before
        passed = None
        for c in [i for i, x in enumerate(parents) if x == node]:
            t = int(tokens[c]) & 0xFFFFFFFF
            ok = t < len(left)
            mass = left[t] / total if ok and total > 0 else 0.0
            rate = (1.0 if draft is None else draft[t]) if ok else 0.0
            if drafts == "distinct" and (rate == 0 or 1 - drawn < 2.0 ** -20):
                continue  # not a draw of this q
            if rate > 0 and float(u[c]) * rate < mass:
                passed = c
                break
            if draft is None:
                if ok:
                    total -= left[t]
                    left[t] = 0
            else:
                left = np.maximum(left / total - draft, 0) if total > 0 else left * 0
                total = left.sum()
                if drafts == "distinct":
                    drawn += positive(q[node])[t]
                    draft = np.where(draft > 0, positive(q[node]) / (1 - drawn) if drawn < 1 else 0.0, 0.0)
                    draft[t] = 0
        if passed is None:
            break
        out.append(int(tokens[passed]))
        path.append(passed)
        node = passed
    if not left.sum() > 0:
        left = target
    c = np.cumsum(left)
    hit = np.nonzero((c > float(u[0]) * c[-1]) & (left > 0))[0]
    last = np.nonzero(left > 0)[0]
    out.append(int(hit[0]) if len(hit) else int(last[-1]) if len(last) else 0)
    return out, path


def run(ctx, seqs, tokens, p, q, u, drafts, ld=None):
    rows = gpu.Rows(ctx, None, [gpu.TreeSeq(0, None, x) for x in seqs])
    ld = ld or rows.deepest
    outs = [torch.full(s, 77, dtype=torch.int32, device="cuda") for s in ((len(seqs), ld), (len(seqs), ld), (len(seqs),))]
    args = [torch.from_numpy(np.ascontiguousarray(x)).cuda() if x is not None else None for x in (tokens, p, q, u)]
    torch.cuda.synchronize()
    gpu.tree_verify(ctx, rows, *args, drafts, *outs)
    ctx.sync()
    return [o.cpu().numpy() for o in outs]


def check(ctx, seqs, tokens, p, q, u, drafts, ld=None):
    out, path, count = run(ctx, seqs, tokens, p, q, u, drafts, ld)
    at, accepted = 0, 0
    for s, parents in enumerate(seqs):
        e = at + len(parents)
        want, way = walk(parents, tokens[at:e], p[at:e], None if q is None else q[at:e], u[at:e], drafts)
        n = len(want)
        assert count[s] == n, (s, drafts)
        assert out[s, :n].tolist() == want and path[s, :n].tolist() == way, (s, drafts, out[s], want, path[s], way)
        assert not out[s, n:].any() and (path[s, n:] == -1).all()
        accepted += n - 1
        at = e
    return accepted


TREES = [[-1], [-1, 0, 1, 2, 3], [-1, 0, 0, 0, 0, 0, 0], [-1, 0, 0, 1, 1, 2, 2, 3, 7, 8], [-1, 0, 0, -2, 2, 2, 2, 5]]


def distributions(rng, rows, vocab, peak=3.0, noise=1.0):
    def softmax(z):
        e = np.exp(z - z.max(axis=1, keepdims=True))
        return (e / e.sum(axis=1, keepdims=True)).astype(np.float32)
    z = rng.standard_normal((rows, vocab)) * peak
    return softmax(z), softmax(z + noise * rng.standard_normal((rows, vocab)))


def drafted(rng, seqs, q, drafts):
    tokens, at = [], 0
    for parents in seqs:
        mine = rng.integers(0, q.shape[1], len(parents))
        for node in range(len(parents)):
            kids = [i for i, x in enumerate(parents) if x == node]
            if not kids:
                continue
            w = q[at + node].astype(np.float64)
            w /= w.sum()
            replace = drafts == "each" or np.count_nonzero(w) < len(kids)
            mine[kids] = (np.argsort(-w)[np.arange(len(kids)) % len(w)] if drafts == "fixed"
                          else rng.choice(len(w), len(kids), replace=replace, p=w))
        tokens += list(mine)
        at += len(parents)
    return np.array(tokens, np.int32)


@pytest.mark.parametrize("vocab", [1, 2, 7, 63, 64, 65, 1000, 4097, 50257])
@pytest.mark.parametrize("drafts", gpu.DRAFTS)
def test_walks_of_every_vocabulary(ctx, drafts, vocab):
    rng = np.random.default_rng(vocab)
    accepted = 0
    for _ in range(4 if vocab > 5000 else 12):
        seqs = [TREES[i] for i in rng.permutation(len(TREES))]
        rows = sum(map(len, seqs))
        p, q = distributions(rng, rows, vocab)
        tokens = drafted(rng, seqs, q, drafts)
        u = rng.random(rows, np.float32)
        accepted += check(ctx, seqs, tokens, p, None if drafts == "fixed" else q, u, drafts, ld=9)
    assert accepted > 0


@pytest.mark.parametrize("drafts", gpu.DRAFTS)
def test_many_children(ctx, drafts):
    """More siblings than are taken at a time, mostly rejected; the same token twice among them."""
    rng = np.random.default_rng(9)
    tree = [-1] + [0] * 600 + [5] * 3
    p, q = distributions(rng, len(tree), 900, peak=1.0, noise=6.0)
    tokens = drafted(rng, [tree], q, drafts)
    tokens[7] = tokens[3]
    tokens[400] = tokens[20]
    for k in range(6):
        u = rng.random(len(tree), np.float32)
        u[1:] = 1 - 0.02 * u[1:] if k < 4 else u[1:]
        if k == 5 and drafts == "fixed":
            u[1:601] = np.float32(1 - 2 ** -24)
        check(ctx, [tree], tokens, p, None if drafts == "fixed" else q, u, drafts)


@pytest.mark.parametrize("drafts", gpu.DRAFTS)
def test_edges(ctx, drafts):
    """Mass on one token, none at all, equal distributions, NaN and negative entries, tokens outside the
    vocabulary, random numbers at both ends."""
    vocab, tree = 130, [-1, 0, 0, 0, 1, 2]
    rng = np.random.default_rng(2)
    p, q = distributions(rng, len(tree), vocab)
    one = np.zeros_like(p)
    one[:, 129] = 1
    bad = p.copy()
    bad[:, 5] = np.nan
    bad[:, 9] = -0.25
    cases = [(one, one), (one, q), (p, one), (np.zeros_like(p), q), (p, p), (bad, q), (p, np.zeros_like(q))]
    for k, (a, b) in enumerate(cases):
        for tokens in (drafted(rng, [tree], q, drafts), np.full(6, 129, np.int32), np.array([0, 3, 3, -1, 200, 7], np.int32)):
            for u in (np.zeros(6, np.float32), np.full(6, 1 - 2.0 ** -24, np.float32), rng.random(6, np.float32)):
                check(ctx, [tree], tokens, a, None if drafts == "fixed" else b, u, drafts)


@pytest.mark.parametrize("drafts", gpu.DRAFTS)
def test_emitted_tokens_have_the_targets_distribution(ctx, drafts):
    """First emitted tokens of 60000 walks: Pearson's statistic over 6 tokens, whose 1 - 1e-6 quantile at 5
    degrees of freedom is 37."""
    vocab, n = 6, 60000
    rng = np.random.default_rng(31)
    p, q = distributions(rng, 1, vocab, peak=1.0)
    tree = [-1, 0, 0]
    seqs = [tree] * 20000
    for chunk in range(n // 20000):
        P, Q = np.repeat(p, 60000, 0), np.repeat(q, 60000, 0)
        tokens = np.zeros((20000, 3), np.int32)
        w = q[0].astype(np.float64) / q[0].astype(np.float64).sum()
        if drafts == "fixed":
            tokens[:, 1:] = np.argsort(-w)[:2]
        else:
            first = rng.choice(vocab, 20000, p=w)
            tokens[:, 1] = first
            if drafts == "each":
                tokens[:, 2] = rng.choice(vocab, 20000, p=w)
            else:
                for t in range(vocab):
                    r = w.copy()
                    r[t] = 0
                    at = np.nonzero(first == t)[0]
                    tokens[at, 2] = rng.choice(vocab, len(at), p=r / r.sum())
        u = rng.random(60000, np.float32)
        out, _, _ = run(ctx, seqs, tokens.ravel(), P, None if drafts == "fixed" else Q, u, drafts)
        counts = np.bincount(out[:, 0], minlength=vocab) if chunk == 0 else counts + np.bincount(out[:, 0], minlength=vocab)
    want = p[0].astype(np.float64) / p[0].sum() * n
    assert ((counts - want) ** 2 / want).sum() < 37, (counts, want)


def test_greedy_walk(ctx):
    rng = np.random.default_rng(6)
    for _ in range(20):
        seqs = [TREES[i] for i in rng.permutation(len(TREES))] + [[-1] + [0] * 150]
        n = sum(map(len, seqs))
        tokens, argmax = rng.integers(0, 3, n).astype(np.int32), rng.integers(0, 3, n).astype(np.int32)
        rows = gpu.Rows(ctx, None, [gpu.TreeSeq(0, None, x) for x in seqs])
        outs = [torch.full(s, 77, dtype=torch.int32, device="cuda") for s in ((6, 12), (6, 12), (6,))]
        t, a = torch.from_numpy(tokens).cuda(), torch.from_numpy(argmax).cuda()
        torch.cuda.synchronize()
        gpu.tree_accept(ctx, rows, t, a, *outs)
        ctx.sync()
        out, path, count = (o.cpu().numpy() for o in outs)
        at = 0
        for s, parents in enumerate(seqs):
            node, want, way = 0, [], []
            while node is not None:
                way.append(node)
                want.append(argmax[at + node])
                node = next((i for i, x in enumerate(parents) if x == node and tokens[at + i] == want[-1]), None)
            k = len(want)
            assert count[s] == k and out[s, :k].tolist() == want and path[s, :k].tolist() == way
            assert not out[s, k:].any() and (path[s, k:] == -1).all()
            at += len(parents)


@pytest.mark.parametrize("drafts", gpu.DRAFTS)
def test_trees_that_leave_the_lds(ctx, drafts):
    """More rows than a workgroup holds, beside a small tree; a chain of as many."""
    rng = np.random.default_rng(12)
    big = [-1] + [int(x) for x in rng.integers(0, np.arange(1, 1500) // 8 + 1)]
    for tree in (big, list(range(-1, 1200))):
        seqs = [TREES[3], tree, TREES[1]]
        rows = sum(map(len, seqs))
        p, q = distributions(rng, rows, 301, peak=1.0, noise=0.5)
        tokens = drafted(rng, seqs, q, drafts)
        for _ in range(3):
            check(ctx, seqs, tokens, p, None if drafts == "fixed" else q, rng.random(rows, np.float32), drafts)
