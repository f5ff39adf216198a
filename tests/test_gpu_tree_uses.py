"""Rows over paged caches as programs use them: whole steps of tree
speculation layer by layer, captured and replayed, on other streams, from two
contexts at once, far into a large cache; and their refusals, after which
nothing has changed."""
import threading

import numpy as np
import pytest
import torch

from ferrolm_amd import gpu
from test_gpu_tree import TREES, Case, attention64, bound, check_attention, cuda, held, sees
from test_gpu_tree_verify import distributions, drafted, walk

pytestmark = pytest.mark.gpu


def outputs(seqs, ld):
    return [torch.zeros(s, dtype=torch.int32, device="cuda") for s in ((seqs, ld), (seqs, ld), (seqs,))]


@pytest.mark.parametrize("fmt", gpu.KV_FORMATS)
def test_steps_of_tree_speculation(ctx, fmt):
    """Three steps over two layers: write, attend, verify, commit, and the next step's rows behind what was
    accepted; everything against numpy, which keeps its own caches."""
    heads, kv_heads, hd, layers, vocab, tree = 6, 2, 64, 2, 97, TREES["deep"]
    rng = np.random.default_rng(3)
    lengths, n = [5, 30, 64], len(tree)
    tables = [[7, 1, 2, 9], [0, 3, 12, 4, 5], [6, 8, 10, 11, 13, 14, 15]]
    kv = gpu.KvCache(ctx, gpu.CacheShape(layers, kv_heads, hd), 16, format=fmt)
    mine = [[[np.zeros((0, kv_heads, hd), np.float32) for _ in range(2)] for _ in range(3)] for _ in range(layers)]

    def write(rows, parts):
        for layer in range(layers):
            x = [[rng.standard_normal((p, kv_heads, hd)).astype(np.float32) for p in parts] for _ in range(2)]
            k, v = (cuda(np.concatenate(y)) for y in x)
            torch.cuda.synchronize()
            gpu.kv_append(ctx, rows, kv, layer, k, v)
            ctx.sync()
            for s in range(3):
                mine[layer][s] = [np.concatenate([mine[layer][s][i], held(x[i][s], fmt)]) for i in range(2)]

    write(gpu.Rows(ctx, kv, [gpu.TreeSeq(0, t, m) for t, m in zip(tables, lengths)], heads=heads), lengths)
    rows = gpu.Rows(ctx, kv, [], heads=heads)
    assert rows.total == 0
    for step in range(3):
        rows.set([gpu.TreeSeq(m, t, tree) for t, m in zip(tables, lengths)])
        write(rows, [n] * 3)
        for layer in range(layers):
            q = rng.standard_normal((3 * n, heads, hd)).astype(np.float32)
            qd, out = cuda(q), torch.empty(3 * n, heads, hd, device="cuda")
            torch.cuda.synchronize()
            gpu.tree_attention(ctx, rows, kv, layer, qd, out)
            ctx.sync()
            for s in range(3):
                want, tol = attention64(q[s * n:s * n + n], *mine[layer][s], sees(lengths[s], tree), fmt)
                assert (np.abs(out.cpu().numpy()[s * n:s * n + n] - want) <= tol).all()
        drafts = gpu.DRAFTS[step]
        p, qq = distributions(rng, 3 * n, vocab, peak=1.5, noise=0.4)
        tokens, u = drafted(rng, [tree] * 3, qq, drafts), rng.random(3 * n, np.float32)
        out, path, count = outputs(3, rows.deepest)
        args = [cuda(tokens), cuda(p), None if drafts == "fixed" else cuda(qq), cuda(u)]
        torch.cuda.synchronize()
        gpu.tree_verify(ctx, rows, *args, drafts, out, path, count)
        gpu.kv_commit(ctx, rows, kv, path, count)
        ctx.sync()
        for s in range(3):
            r = slice(s * n, s * n + n)
            want, way = walk(tree, tokens[r], p[r], None if drafts == "fixed" else qq[r], u[r], drafts)
            assert int(count[s]) == len(want) and out[s, :len(want)].tolist() == want
            assert path[s, :len(way)].tolist() == way
            for layer in range(layers):
                mine[layer][s] = [np.concatenate([x[:lengths[s]], x[[lengths[s] + i for i in way]]]) for x in mine[layer][s]]
            lengths[s] += len(way)
        whole = gpu.Rows(ctx, kv, [gpu.TreeSeq(m, t, 0) for t, m in zip(tables, lengths)])
        for layer in range(layers):
            k, v = (torch.empty(whole.tokens, kv_heads, hd, device="cuda") for _ in range(2))
            torch.cuda.synchronize()
            gpu.kv_gather(ctx, whole, kv, layer, k, v)
            ctx.sync()
            for i, have in enumerate((k, v)):
                bad = have.cpu().numpy() != np.concatenate([mine[layer][s][i] for s in range(3)])
                assert not bad.any(), (step, layer, i, np.unique(np.argwhere(bad)[:, 0]))


def test_two_captured_graphs_and_eager_calls(ctx):
    """Write, attention and verification captured behind another stream's work, twice with rows of their own;
    replayed in turn with new inputs and eager calls in between, every replay against the eager result."""
    heads, kv_heads, hd, vocab = 8, 2, 128, 1000
    cases = [Case(ctx, "int8", kv_heads, hd, [(700, TREES["deep"]), (33, TREES["fan"])], seed=1),
             Case(ctx, "int8", kv_heads, hd, [(260, TREES["chain"])], seed=2)]
    side = torch.cuda.Stream()
    ctx.wait(side)
    ctx.signal(side)
    made = []
    for c in cases:
        c.fill()
        rows, n = c.rows(heads), sum(len(p) for p in c.parents)
        x = torch.randn(n, heads + 2 * kv_heads, hd, device="cuda")
        p = torch.softmax(torch.randn(n, vocab, device="cuda"), 1)
        tokens = torch.randint(0, 20, (n,), dtype=torch.int32, device="cuda")
        u = torch.rand(n, device="cuda")
        out = torch.empty(n, heads, hd, device="cuda")
        res = outputs(len(c.pos), rows.deepest)
        back = [torch.empty(n, kv_heads, hd, device="cuda") for _ in range(2)]

        def work(c=c, rows=rows, x=x, p=p, tokens=tokens, u=u, out=out, res=res, back=back):
            y = x * 2.0  # the other stream's work before, and after
            ctx.wait(torch.cuda.current_stream())
            gpu.kv_append(ctx, rows, c.kv, 0, y[:, heads:heads + kv_heads], y[:, heads + kv_heads:])
            gpu.kv_gather(ctx, rows, c.kv, 0, *back, context=False)
            gpu.tree_attention(ctx, rows, c.kv, 0, y[:, :heads], out)
            gpu.tree_verify(ctx, rows, tokens, p, None, u, "fixed", *res)
            ctx.signal(torch.cuda.current_stream())
            return out + 0.0, *(r + 0 for r in res), *(b + 0.0 for b in back)

        with torch.cuda.stream(side):
            work()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            got = work()
        made.append((g, got, work, x, u))
    torch.cuda.synchronize()
    for turn in range(4):
        for g, got, work, x, u in made:
            x.copy_(torch.randn_like(x))
            u.copy_(torch.rand_like(u))
            torch.cuda.synchronize()
            g.replay()
        torch.cuda.synchronize()
        kept = [[t.clone() for t in got] for _, got, _, _, _ in made]
        for (g, got, work, x, u), k in zip(made, kept):
            with torch.cuda.stream(side):
                want = work()
            torch.cuda.synchronize()
            for a, b in zip(k, want):
                assert torch.equal(a, b), turn


def test_rows_are_not_planned_into_a_capture(ctx):
    c = Case(ctx, "int8", 1, 64, [(20, 2)], seed=3)
    rows = c.rows(1)
    side = torch.cuda.Stream()
    ctx.wait(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        ctx.wait(torch.cuda.current_stream())
        with pytest.raises(gpu.FgError, match="captured"):
            rows.set([gpu.TreeSeq(20, c.tables[0], 1)])
        with pytest.raises(gpu.FgError, match="captured"):
            c.rows(1)
        ctx.signal(torch.cuda.current_stream())
    assert rows.total == 2
    rows.set([gpu.TreeSeq(20, c.tables[0], 1)])
    assert rows.total == 1


def test_inputs_and_outputs_of_another_stream(ctx):
    """Queries made late on a busy stream, and read on it, with no synchronisation between."""
    c = Case(ctx, "fp8", 2, 64, [(900, 4)], seed=5)
    c.fill()
    rows = c.rows(4)
    q = torch.randn(4, 4, 64, device="cuda")
    want = torch.empty_like(q)
    torch.cuda.synchronize()
    gpu.tree_attention(ctx, rows, c.kv, 0, q, want)
    ctx.sync()
    side = torch.cuda.Stream()
    big = torch.randn(4096, 4096, device="cuda")
    for _ in range(3):
        late, out = torch.zeros_like(q), torch.zeros_like(q)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            y = big
            for _ in range(6):
                y = y @ big * 1e-3
            late.copy_(q)
            ctx.wait(side)
            gpu.tree_attention(ctx, rows, c.kv, 0, late, out)
            ctx.signal(side)
            got = out.clone()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_two_contexts_at_once(ctx):
    """Two host threads with a context each over one cache, against the same calls alone."""
    c = Case(ctx, "int8", 2, 128, [(1500, TREES["deep"]), (800, 3)], seed=6)
    c.fill()
    other = gpu.Context(0)
    q = torch.randn(13, 8, 128, device="cuda")
    p = torch.softmax(torch.randn(13, 5000, device="cuda") * 2, 1)
    tok, u = torch.randint(0, 50, (13,), dtype=torch.int32, device="cuda"), torch.rand(13, device="cuda")
    torch.cuda.synchronize()
    results = {}

    def run(x, name):
        rows = gpu.Rows(x, c.kv, [gpu.TreeSeq(n, t, par) for n, t, par in zip(c.pos, c.tables, c.parents)], heads=8)
        outs = []
        for _ in range(40):
            out, res = torch.zeros(13, 8, 128, device="cuda"), outputs(2, rows.deepest)
            torch.cuda.synchronize()
            gpu.tree_attention(x, rows, c.kv, 0, q, out)
            gpu.tree_verify(x, rows, tok, p, None, u, "fixed", *res)
            x.sync()
            outs.append([out, *res])
        results[name] = outs
        rows.close()

    run(ctx, "alone")
    threads = [threading.Thread(target=run, args=(x, n)) for x, n in ((ctx, "a"), (other, "b"))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for name in ("a", "b"):
        assert len(results[name]) == 40
        for one in results[name]:
            for x, y in zip(one, results["alone"][0]):
                assert torch.equal(x, y)
    other.close()


@pytest.mark.parametrize("fmt", ["int8", "f32"])
def test_blocks_behind_the_first_4_gib(ctx, fmt):
    heads, kv_heads, hd = 8, 8, 128
    per = kv_heads * (32 * hd + 128 if fmt == "int8" else 64 * hd)
    blocks = ((9 << 29) if fmt == "int8" else (9 << 30)) // per + 40
    c = Case(ctx, fmt, kv_heads, hd, [(100, TREES["deep"])], seed=7)
    c.kv = gpu.KvCache(ctx, gpu.CacheShape(1, kv_heads, hd), blocks, format=fmt)
    c.tables = [np.array([blocks - 1 - 3 * i for i in range(7)], np.uint32)]
    c.fill()
    rows = c.rows(heads)
    k, v = (torch.empty(110, kv_heads, hd, device="cuda") for _ in range(2))
    q = c.rng.standard_normal((10, heads, hd)).astype(np.float32)
    qd, out = cuda(q), torch.empty(10, heads, hd, device="cuda")
    torch.cuda.synchronize()
    gpu.kv_gather(ctx, rows, c.kv, 0, k, v)
    gpu.tree_attention(ctx, rows, c.kv, 0, qd, out)
    ctx.sync()
    hk, hv = held(c.k[0], fmt), held(c.v[0], fmt)
    assert np.array_equal(k.cpu().numpy(), hk) and np.array_equal(v.cpu().numpy(), hv)
    want, tol = attention64(q, hk, hv, sees(100, TREES["deep"]), fmt)
    assert (np.abs(out.cpu().numpy() - want) <= tol).all()
    c.kv.close()


def test_refusals_leave_everything_as_it_was(ctx):
    c = Case(ctx, "int8", 2, 64, [(20, TREES["deep"])], seed=8)
    c.fill()
    rows, n, blocks = c.rows(4), 10, c.kv.blocks
    before = c.kv.layer(0)
    k = torch.zeros(n, 2, 64, device="cuda")
    q, out = torch.zeros(n, 4, 64, device="cuda"), torch.full((n, 4, 64), 3.0, device="cuda")
    p, tok, u = torch.zeros(n, 33, device="cuda"), torch.zeros(n, dtype=torch.int32, device="cuda"), torch.zeros(n, device="cuda")
    res = outputs(1, rows.deepest)
    torch.cuda.synchronize()
    other = gpu.Context(0)
    shape = gpu.KvCache(ctx, gpu.CacheShape(1, 2, 32), 40)
    small = gpu.KvCache(ctx, gpu.CacheShape(1, 2, 64), 1, format="int8")
    T = gpu.TreeSeq
    for call, match in (
            (lambda: gpu.Rows(ctx, c.kv, [T(20, c.tables[0], 40)], heads=4), "overrun"),
            (lambda: gpu.Rows(ctx, c.kv, [T(0, [blocks], 3)], heads=4), "block id beyond"),
            (lambda: gpu.Rows(ctx, c.kv, [T(0, None, 3)], heads=4), "without a block table"),
            (lambda: gpu.Rows(ctx, c.kv, [T(-1, c.tables[0], 3)], heads=4), "negative"),
            (lambda: gpu.Rows(ctx, c.kv, [T(0, c.tables[0], [-1, 1])], heads=4), "earlier row"),
            (lambda: gpu.Rows(ctx, c.kv, [T(0, c.tables[0], [-3])], heads=4), "earlier row"),
            (lambda: gpu.Rows(ctx, c.kv, [T(0, c.tables[0], [-2, 0])], heads=4), "no children"),
            (lambda: gpu.Rows(ctx, c.kv, [T(0, c.tables[0], 3)], heads=3), "multiple of the kv heads"),
            (lambda: gpu.Rows(ctx, c.kv, [T(0, c.tables[0], 3)], heads=600), "GQA group"),
            (lambda: gpu.Rows(ctx, None, [T(0, None, [-1] + [0] * 4096)]), "at most 4096"),
            (lambda: gpu.KvCache(ctx, gpu.CacheShape(1, 2, 96), 4, format="fp8"), "head_dim 96"),
            (lambda: gpu.tree_attention(other, rows, c.kv, 0, q, out), "another context"),
            (lambda: gpu.tree_attention(ctx, rows, c.kv, 1, q, out), "no such layer"),
            (lambda: gpu.kv_append(ctx, rows, small, 0, k, k), "block id beyond"),
            (lambda: gpu.check(gpu.lib().fg_kv_append(ctx.h, rows.h, shape.h, 0, k.data_ptr(), k.data_ptr(), 128)),
             "another cache shape"),
            (lambda: gpu.check(gpu.lib().fg_tree_attention(ctx.h, rows.h, c.kv.h, 0, q.data_ptr() + 4, 256,
                                                           out.data_ptr(), 256)), "aligned"),
            (lambda: gpu.check(gpu.lib().fg_tree_attention(ctx.h, rows.h, c.kv.h, 0, q.data_ptr(), 252,
                                                           out.data_ptr(), 256)), "far apart"),
            (lambda: gpu.check(gpu.lib().fg_tree_attention(ctx.h, rows.h, c.kv.h, 0, None, 256, out.data_ptr(), 256)),
             "null array"),
            (lambda: gpu.tree_verify(ctx, rows, tok, p, None, u, "each", *res), "come with q"),
            (lambda: gpu.check(gpu.lib().fg_tree_verify(ctx.h, rows.h, 2, (1 << 30) + 4, tok.data_ptr(), p.data_ptr(), None,
                                                        u.data_ptr(), *(r.data_ptr() for r in res), rows.deepest)), "2.30 tokens"),
            (lambda: gpu.tree_verify(ctx, rows, tok, p, p, u, "fixed", *res), "come with q"),
            (lambda: gpu.tree_verify(ctx, rows, tok, p, None, u, "fixed", *outputs(1, rows.deepest - 1)), "longest branch"),
            (lambda: gpu.tree_accept(ctx, gpu.Rows(ctx, None, [T(0, None, [-1, -1])]), tok[:2], tok[:2], *outputs(1, 3)),
             "root of its others"),
            (lambda: gpu.tree_accept(ctx, gpu.Rows(ctx, None, [T(0, None, 0)]), tok[:0], tok[:0], *outputs(1, 3)),
             "root of its others")):
        with pytest.raises(gpu.FgError, match=match):
            call()
    for call, match in (
            (lambda: gpu.tree_attention(ctx, rows, c.kv, 0, q.half(), out), "expected"),
            (lambda: gpu.tree_attention(ctx, rows, c.kv, 0, q[:5], out), "expected"),
            (lambda: gpu.tree_attention(ctx, rows, c.kv, 0, q.cpu(), out), "on cpu"),
            (lambda: gpu.tree_attention(ctx, rows, c.kv, 0, q.transpose(1, 2).contiguous().transpose(1, 2), out), "dense"),
            (lambda: gpu.kv_append(ctx, gpu.Rows(ctx, None, [T(0, None, 2)]), c.kv, 0, k, k), "without a cache"),
            (lambda: gpu.tree_verify(ctx, rows, tok, p, None, u, "some", *res), "one of"),
            (lambda: gpu.KvCache(ctx, gpu.CacheShape(1, 2, 64), 4, format="int4"), "one of")):
        with pytest.raises(ValueError, match=match):
            call()
    ctx.sync()
    for a, b in zip(before, c.kv.layer(0)):
        assert np.array_equal(a, b)
    assert (out == 3.0).all() and not any(r.any() for r in res)
    # a refused plan leaves the one before
    with pytest.raises(gpu.FgError, match="overrun"):
        rows.set([T(20, c.tables[0], 60)])
    gpu.tree_attention(ctx, rows, c.kv, 0, q, out)
    ctx.sync()
    want = np.array([held(c.v[0], "int8").astype(np.float64)[m].mean(0) for m in sees(20, TREES["deep"])])
    assert rows.total == n  # q = 0: the mean of the values that a row sees
    assert np.abs(out.cpu().numpy() - want.repeat(2, 1)).max() <= bound(0, 0, 30, 1) * np.abs(c.v[0]).max()
    other.close()


def test_rows_outlive_their_context_to_be_closed_only():
    x = gpu.Context(0)
    kv = gpu.KvCache(x, gpu.CacheShape(1, 1, 64), 4, format="int8")
    rows = gpu.Rows(x, kv, [gpu.TreeSeq(0, [1], 2)])
    k = torch.zeros(2, 1, 64, device="cuda")
    x.close()
    with pytest.raises(ValueError, match="closed"):
        rows.set([gpu.TreeSeq(0, [1], 1)])
    with pytest.raises(gpu.FgError, match="null"):
        gpu.kv_append(x, rows, kv, 0, k, k)
    rows.close()


def test_nothing_to_do(ctx):
    c = Case(ctx, "fp8", 1, 64, [(3, 1)], seed=9)
    rows = gpu.Rows(ctx, c.kv, [gpu.TreeSeq(0, None, 0), gpu.TreeSeq(3, c.tables[0], 0)], heads=2)
    assert (rows.total, rows.tokens, rows.deepest) == (0, 3, 0)
    none = torch.empty(0, 1, 64, device="cuda")
    gpu.kv_append(ctx, rows, c.kv, 0, none, none)
    gpu.tree_attention(ctx, rows, c.kv, 0, torch.empty(0, 2, 64, device="cuda"), torch.empty(0, 2, 64, device="cuda"))
    k, v = (torch.ones(3, 1, 64, device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    gpu.kv_gather(ctx, rows, c.kv, 0, k, v)  # what the cleared cache holds
    ctx.sync()
    assert not k.any() and not v.any()


def test_gather_of_sequences_without_rows(ctx):
    """Beside shorter ones with rows, and alone."""
    c = Case(ctx, "int8", 2, 32, [(75, 0), (5, 2), (0, 0), (30, 0)], seed=10)
    c.fill()
    for seqs in ([0, 1, 2, 3], [0, 3], [3]):
        rows = gpu.Rows(ctx, c.kv, [gpu.TreeSeq(c.pos[s], c.tables[s], c.parents[s]) for s in seqs])
        k, v = (torch.zeros(rows.tokens, 2, 32, device="cuda") for _ in range(2))
        torch.cuda.synchronize()
        gpu.kv_gather(ctx, rows, c.kv, 0, k, v)
        ctx.sync()
        assert np.array_equal(k.cpu().numpy(), held(np.concatenate([c.k[s] for s in seqs]), "int8"))
        assert np.array_equal(v.cpu().numpy(), held(np.concatenate([c.v[s] for s in seqs]), "int8"))


@pytest.mark.parametrize("fmt", gpu.KV_FORMATS)
@pytest.mark.parametrize("sign", [-1, 1])
def test_scores_of_any_size(ctx, fmt, sign):
    """Scores of +-8e32, all alike: the mean of the values, over waves, parts and pages."""
    c = Case(ctx, fmt, 2, 64, [(3000, 3), (20, TREES["fan"])], seed=11)
    for k in c.k:
        k[:] = 1e16 * sign
    c.fill()
    q = np.full((8, 4, 64), 1e16, np.float32)
    qd, out = cuda(q), torch.empty(8, 4, 64, device="cuda")
    torch.cuda.synchronize()
    gpu.tree_attention(ctx, c.rows(4), c.kv, 0, qd, out)
    ctx.sync()
    at = 0
    for n, p, v in zip(c.pos, c.parents, c.v):
        v = held(v, fmt).astype(np.float64)
        for i, m in enumerate(sees(n, p)):
            err = np.abs(out[at + i].cpu().numpy() - v[m].mean(0).repeat(2, 0))
            assert (err <= bound(0, 0, m.sum(), 2.5) * np.abs(v[m]).mean(0).repeat(2, 0)).all()
        at += len(p)


@pytest.mark.parametrize("fmt,heads,kv_heads,hd,tree", [
    ("int8", 16, 8, 128, "deep"), ("fp8", 8, 8, 64, "fan"), ("int8", 8, 8, 128, "one"), ("f32", 32, 8, 32, "forest"),
    ("fp8", 256, 8, 128, "deep"), ("f32", 16, 8, 64, "one")])
@pytest.mark.parametrize("seqs", [12, 40, 70])
def test_batches_around_what_the_card_holds(ctx, fmt, heads, kv_heads, hd, tree, seqs):
    """Contexts in pieces of their own, in pieces that share a workgroup with others', and whole: fewer sequences
    than there are places for a kv head (32), somewhat more, and many more, some of them without rows."""
    rng = np.random.default_rng(seqs)
    lens = np.exp(rng.uniform(0, np.log(700), seqs)).astype(int)
    c = Case(ctx, fmt, kv_heads, hd, [(int(n), [] if i % 11 == 5 else TREES[tree]) for i, n in enumerate(lens)], seed=seqs)
    c.fill()
    check_attention(c, heads)


@pytest.mark.parametrize("fmt,hd,rows", [("int8", 64, 40), ("f32", 16, 1)])
def test_pieces_end_at_their_most_pages(ctx, fmt, hd, rows):
    """A context of more pages than a piece holds for each of the two workgroups of a kv head: a workgroup's next
    piece goes on in it. Its blocks repeat; three of 128 heads are compared."""
    kv_heads, distinct, pages = 128, 48, 2300
    c = Case(ctx, fmt, kv_heads, hd, [(distinct * 16, rows)], seed=12)
    c.fill()
    first = c.tables[0][:distinct]
    table = np.concatenate([np.resize(first, pages), c.tables[0][distinct:]])
    seen = gpu.Rows(ctx, c.kv, [gpu.TreeSeq(pages * 16, table, rows)], heads=kv_heads)
    q = c.rng.standard_normal((rows, kv_heads, hd)).astype(np.float32)
    qd, out = cuda(q), torch.empty(rows, kv_heads, hd, device="cuda")
    torch.cuda.synchronize()
    gpu.tree_attention(ctx, seen, c.kv, 0, qd, out)
    ctx.sync()
    got, some = out.cpu().numpy(), [0, 77, 127]
    at = np.concatenate([np.resize(np.arange(distinct * 16), pages * 16), distinct * 16 + np.arange(rows)])
    k, v = (held(x[0][:, some], fmt)[at] for x in (c.k, c.v))
    pick = [0, rows - 1]
    want, tol = attention64(q[pick][:, some], k, v, sees(pages * 16, list(range(-1, rows - 1)))[pick], fmt)
    assert (np.abs(got[pick][:, some] - want) <= tol).all()


@pytest.mark.parametrize("fmt", gpu.KV_FORMATS)
@pytest.mark.parametrize("size", [1e-18, 1e-6, 1e6])
def test_values_of_any_size(ctx, fmt, size):
    """The weights' bits do not depend on the size of the values; a context that begins with zeros, and one whose
    values grow to it."""
    c = Case(ctx, fmt, 2, 64, [(900, TREES["deep"]), (70, 1), (300, 4)], seed=13)
    for v in c.v:
        v *= np.float32(size)
    c.v[0][:300] = 0
    c.v[2][:300] *= np.geomspace(1e-3, 1, 300, dtype=np.float32)[:, None, None]
    c.fill()
    check_attention(c, 8)
