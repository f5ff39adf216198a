"""Rows over paged caches on the device (fg_kv_append, fg_kv_gather,
fg_kv_commit, fg_tree_attention) against plain 64-bit forms: every cache
format and head layout, contexts from nothing to thousands of tokens, chains,
trees and unused rows, strided inputs, masked places that hold NaN.

Tolerances. The quantizer is defined bit for bit. For the attention, with
eps = 2^-24 (half a step of f32): scores are sums of products with the query
split to 2^-21 (f32 keys likewise, whose cross term of 2^-22 is dropped)
through at most 16 dependent f32 sums, so a score is off by at most
d = (2^-21 c + 16 eps) sum|q k| / sqrt(hd), c = 1 for 8-bit codes (exact in
f16) and 2.5 for f32 keys. A probability is then off by 2 d (its own and its
sum's), by the exponential (2^-22) and the rounding of its argument (2 eps of
the largest score, in log 2 units); the weight by its split (2^-21, and f32
values by theirs, 1.5 x 2^-21); the sums over n tokens by at most n / 4 + 64
dependent additions. The output is off by sum p |v| times the sum of these.
That is relative to each weight. A weight (p times its value's scale s, against
codes up to c) is held to 2^-25 where that is more, half of f16's smallest
step, while the largest of its sum is 2^9 at least: n such errors times c are
n c 2^-34 of the largest p s, and c s is the largest |v| of its row: 2^-34 n
max(p max|v|) more, which shows where the token that has nearly all weight has
a zero in a channel."""
import numpy as np
import pytest
import torch

from ferrolm_amd import gpu

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -24
E4M3 = torch.float8_e4m3fn


def quantized(x, fmt):
    """(codes as numbers, scales) of rows along the last axis: the definition in f32 steps (numpy)."""
    x = np.asarray(x, np.float32)
    if fmt == "f32":
        return x, np.ones(x.shape[:-1] + (1,), np.float32)
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        s = np.abs(x).max(axis=-1, keepdims=True) * (np.float32(1) / np.float32(127 if fmt == "int8" else 448))
        s = np.where(np.isfinite(x).all(axis=-1, keepdims=True), s, np.float32(np.nan)).astype(np.float32)
        y = np.where(s > 0, x / s, np.float32(0)).astype(np.float32)
        if fmt == "int8":
            return np.clip(np.rint(y), -127, 127).astype(np.float32), s
        y = np.clip(y, -448, 448)
        return torch.from_numpy(y).to(E4M3).float().numpy(), s


def held(x, fmt):
    """The f32 values that a cache holds for x."""
    c, s = quantized(x, fmt)
    with np.errstate(invalid="ignore"):
        return (c * s).astype(np.float32)


def cuda(x):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


class Case:
    """Sequences over a cache of shuffled blocks, filled with random keys and values."""

    def __init__(self, ctx, fmt, kv_heads, hd, seqs, seed=0, layers=1, layer=0):
        """seqs: (cached tokens, parents) each."""
        rng = np.random.default_rng(seed)
        self.ctx, self.fmt, self.kv_heads, self.hd, self.layer = ctx, fmt, kv_heads, hd, layer
        self.parents = [list(range(-1, p - 1)) if isinstance(p, int) else list(p) for _, p in seqs]
        self.pos = [n for n, _ in seqs]
        need = [(n + len(p) + 15) // 16 for n, p in zip(self.pos, self.parents)]
        order = rng.permutation(sum(need) + 3).astype(np.uint32)
        ends = np.cumsum(need)
        self.tables = [order[e - n:e] for e, n in zip(ends, need)]
        self.kv = gpu.KvCache(ctx, gpu.CacheShape(layers, kv_heads, hd), sum(need) + 3, format=fmt)
        self.k, self.v = [], []
        for n, p in zip(self.pos, self.parents):
            shape = (n + len(p), kv_heads, hd)
            self.k.append((rng.standard_normal(shape) * np.exp(0.5 * rng.standard_normal(shape[:2] + (1,)))).astype(np.float32))
            self.v.append((rng.standard_normal(shape) * np.exp(0.5 * rng.standard_normal(shape[:2] + (1,)))).astype(np.float32))
        self.rng = rng

    def fill(self):
        whole = gpu.Rows(self.ctx, self.kv, [gpu.TreeSeq(0, t, len(k)) for t, k in zip(self.tables, self.k)])
        torch.cuda.synchronize()
        gpu.kv_append(self.ctx, whole, self.kv, self.layer, cuda(np.concatenate(self.k)), cuda(np.concatenate(self.v)))
        self.ctx.sync()

    def rows(self, heads=None, chains=False):
        return gpu.Rows(self.ctx, self.kv, [gpu.TreeSeq(n, t, len(p) if chains else p)
                                            for n, t, p in zip(self.pos, self.tables, self.parents)], heads=heads)


def sees(n, parents):
    """[rows][n + rows]"""
    m = np.zeros((len(parents), n + len(parents)), bool)
    for i, p in enumerate(parents):
        if p == -2:
            continue
        m[i, :n] = True
        if p >= 0:
            m[i, n:] = m[p, n:]
        m[i, n + i] = True
    return m


def attention64(q, k, v, visible, fmt):
    """(output, bound of sum p |v| x error) of q [rows][heads][hd] over k, v [tokens][kv_heads][hd]."""
    rows, heads, hd = q.shape
    c = 2.5 if fmt == "f32" else 1.0
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    q, k, v = q.astype(np.float64), k.astype(np.float64), v.astype(np.float64)
    for h in range(heads):
        kh, vh = k[:, h * k.shape[1] // heads], v[:, h * k.shape[1] // heads]
        for r in range(rows):
            m = visible[r]
            if not m.any():
                continue
            s = kh[m] @ q[r, h] / np.sqrt(hd)
            w = np.exp(s - s.max())
            w /= w.sum()
            out[r, h] = w @ vh[m]
            spread = (np.abs(kh[m]) @ np.abs(q[r, h])).max() / np.sqrt(hd)
            tol[r, h] = w @ np.abs(vh[m]) * bound(spread, np.abs(s).max(), m.sum(), c)
            tol[r, h] += 2.0 ** -34 * m.sum() * (w * np.abs(vh[m]).max(axis=1)).max()
    return out, tol


def bound(spread, top, n, c):
    d = (2.0 ** -21 * c + 16 * EPS) * spread
    return 2 * d + 2.0 ** -22 + 2 * EPS * 1.4427 * top + 2.5 * 2.0 ** -21 + (n / 4 + 64) * EPS


def check_attention(case, heads, q=None):
    ctx = case.ctx
    total = sum(len(p) for p in case.parents)
    if q is None:
        q = case.rng.standard_normal((total, heads, case.hd)).astype(np.float32)
    out = torch.full((total, heads, case.hd), float("nan"), device="cuda")
    qd = cuda(q)
    rows = case.rows(heads)
    torch.cuda.synchronize()
    gpu.tree_attention(ctx, rows, case.kv, case.layer, qd, out)
    ctx.sync()
    got = out.cpu().numpy()
    at = 0
    for n, p, k, v in zip(case.pos, case.parents, case.k, case.v):
        want, tol = attention64(q[at:at + len(p)], held(k, case.fmt), held(v, case.fmt), sees(n, p), case.fmt)
        have = got[at:at + len(p)]
        bad = ~(np.abs(have - want) <= tol)
        assert not bad.any(), (case.fmt, n, len(p), np.abs(have - want).max(), np.argwhere(bad)[:3], tol.max())
        at += len(p)
    return got


TREES = {"one": [-1], "chain": [-1, 0, 1, 2, 3], "fan": [-1, 0, 0, 0, 0], "deep": [-1, 0, 0, 1, 1, 2, 2, 3, 7, 8],
         "forest": [-1, -1, -1, 0, 1, 2], "unused": [-1, 0, -2, 0, -2, 1, 5], "none": [-2, -2]}
LAYOUTS = [(1, 1, 16), (6, 2, 16), (4, 4, 32), (12, 3, 32), (9, 3, 64), (32, 32, 64), (16, 1, 64), (8, 2, 128),
           (20, 1, 128), (32, 1, 128), (40, 1, 32)]


# ---------------------------------------------------------------------------
# The cache
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("hd", [16, 32, 64, 128])
@pytest.mark.parametrize("fmt", gpu.KV_FORMATS)
def test_written_rows_read_back_as_defined_and_others_stay(ctx, fmt, hd):
    c = Case(ctx, fmt, 3, hd, [(0, 1), (5, [-1, 0, 0, 1]), (16, 37), (30, [-1, -2, 0, -2, 2]), (15, 2)], seed=hd,
             layers=2, layer=1)
    # special rows: zeros, one far value, a largest value that is subnormal, infinities and NaN, ties of the rounding
    c.k[2][16] = 0
    c.k[2][17] = 0
    c.k[2][17, :, 3] = 1e30
    c.k[2][18] = 1e-42
    c.k[2][19, 0, 1] = np.inf
    c.v[2][20, 1, 2] = np.nan
    c.v[2][21] = (np.arange(hd) % 16 + 0.5) / 8
    c.v[2][21, :, 0] = 127 / 8
    c.v[2][22, 2, 0] = -np.inf
    c.fill()
    before = [x.copy() for x in c.kv.layer(0)]
    # new values for the rows, as columns of a wider matrix
    rows = c.rows()
    total = rows.total
    x = c.rng.standard_normal((total, 8, hd)).astype(np.float32)
    new_k, new_v = x[:, 1:4], x[:, 5:8]
    at = 0
    want = [[k.copy(), v.copy()] for k, v in zip(c.k, c.v)]
    for s, (n, p) in enumerate(zip(c.pos, c.parents)):
        for i, par in enumerate(p):
            if par != -2 and not (s == 2 and i < 7):
                want[s][0][n + i], want[s][1][n + i] = new_k[at + i], new_v[at + i]
            elif s == 2 and i < 7:
                new_k[at + i], new_v[at + i] = want[s][0][n + i], want[s][1][n + i]
        at += len(p)
    d = cuda(x)
    torch.cuda.synchronize()
    gpu.kv_append(ctx, rows, c.kv, 1, d[:, 1:4], d[:, 5:8])
    k, v = (torch.full((rows.tokens, 3, hd), 7.0, device="cuda") for _ in range(2))
    kr, vr = (torch.full((total, 3, hd), 7.0, device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    gpu.kv_gather(ctx, rows, c.kv, 1, k, v)
    gpu.kv_gather(ctx, rows, c.kv, 1, kr, vr, context=False)
    ctx.sync()
    wk, wv = (held(np.concatenate([w[i] for w in want]), fmt) for i in range(2))
    assert np.array_equal(k.cpu().numpy(), wk, equal_nan=True)
    assert np.array_equal(v.cpu().numpy(), wv, equal_nan=True)
    first = np.cumsum([0] + [len(w[0]) for w in want])
    for have, all_ in ((kr, wk), (vr, wv)):
        have = have.cpu().numpy()
        at = 0
        for f, n, p in zip(first, c.pos, c.parents):
            for i, par in enumerate(p):
                assert np.array_equal(have[at], all_[f + n + i] if par != -2 else np.zeros((3, hd)), equal_nan=True)
                at += 1
    # the other layer, and through the host calls
    for a, b in zip(before, c.kv.layer(0)):
        assert np.array_equal(a, b)
    hk, hv = c.kv.layer(1)
    hk, hv = (a.reshape(-1, 3, 16, hd) for a in (hk, hv))
    for s, t in enumerate(c.tables):
        for i in range(len(want[s][0])):
            assert np.array_equal(hk[t[i // 16], :, i % 16], wk[first[s] + i], equal_nan=True)
            assert np.array_equal(hv[t[i // 16], :, i % 16], wv[first[s] + i], equal_nan=True)


@pytest.mark.parametrize("fmt", gpu.KV_FORMATS)
def test_host_write_is_the_same_quantizer(ctx, fmt):
    kv = gpu.KvCache(ctx, gpu.CacheShape(2, 2, 32), 5, format=fmt)
    rng = np.random.default_rng(3)
    k, v = (rng.standard_normal((5 * 2 * 16, 32)).astype(np.float32) for _ in range(2))
    kv.set_layer(1, k, v)
    a, b = kv.layer(1)
    assert np.array_equal(a, held(k, fmt).ravel()) and np.array_equal(b, held(v, fmt).ravel())
    assert not any(x.any() for x in kv.layer(0))


@pytest.mark.parametrize("fmt", gpu.KV_FORMATS)
def test_commit_moves_the_branch(ctx, fmt):
    layers = 3
    c = Case(ctx, fmt, 2, 64, [(13, TREES["deep"]), (0, TREES["deep"]), (31, TREES["fan"]), (5, 1)], seed=5,
             layers=layers)
    held_ = []
    for layer in range(layers):
        c.layer = layer
        c.k = [x + np.float32(layer) for x in c.k]
        c.fill()
        held_.append([(held(k, fmt), held(v, fmt)) for k, v in zip(c.k, c.v)])
    rows = c.rows()
    path = np.full((4, 6), -1, np.int32)
    path[0, :5] = [0, 1, 3, 7, 8]
    path[1, :3] = [0, 2, 6]
    path[2, :2] = [0, 4]
    path[3, :1] = [0]
    count = np.array([5, 3, 2, 1], np.int32)
    p, n = cuda(path), cuda(count)
    torch.cuda.synchronize()
    gpu.kv_commit(ctx, rows, c.kv, p, n)
    for layer in range(layers):
        k, v = (torch.empty(rows.tokens, 2, 64, device="cuda") for _ in range(2))
        torch.cuda.synchronize()
        gpu.kv_gather(ctx, rows, c.kv, layer, k, v)
        ctx.sync()
        at = 0
        for s, (pos, par) in enumerate(zip(c.pos, c.parents)):
            wk, wv = (x.copy() for x in held_[layer][s])
            for j in range(count[s]):
                wk[pos + j], wv[pos + j] = held_[layer][s][0][pos + path[s, j]], held_[layer][s][1][pos + path[s, j]]
            e = at + pos + len(par)
            assert np.array_equal(k[at:e].cpu().numpy(), wk) and np.array_equal(v[at:e].cpu().numpy(), wv)
            at = e


# ---------------------------------------------------------------------------
# Attention
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("heads,kv_heads,hd", LAYOUTS)
@pytest.mark.parametrize("fmt", gpu.KV_FORMATS)
def test_attention_of_every_layout(ctx, fmt, heads, kv_heads, hd):
    c = Case(ctx, fmt, kv_heads, hd, [(0, [-1]), (1, TREES["deep"]), (15, 3), (16, TREES["fan"]), (47, TREES["unused"]),
                                      (130, TREES["forest"])], seed=heads + hd)
    c.fill()
    check_attention(c, heads)


@pytest.mark.parametrize("tree", list(TREES))
@pytest.mark.parametrize("n", [0, 1, 17, 31, 300])
def test_attention_of_every_tree(ctx, n, tree):
    c = Case(ctx, "int8", 2, 64, [(n, TREES[tree])], seed=n)
    c.fill()
    got = check_attention(c, 4)
    for i, p in enumerate(TREES[tree]):
        if p == -2:
            assert not got[i].any()


@pytest.mark.parametrize("fmt", gpu.KV_FORMATS)
@pytest.mark.parametrize("n,rows", [(0, 70), (9, 33), (100, 129), (1000, 1), (5000, 2), (3, 300)])
def test_attention_of_chains(ctx, fmt, n, rows):
    c = Case(ctx, fmt, 2, 64 if rows > 2 else 128, [(n, rows)], seed=n + rows)
    c.fill()
    check_attention(c, 6)


def test_attention_of_ragged_batches(ctx):
    rng = np.random.default_rng(1)
    seqs = [(int(rng.integers(0, 900)), list(TREES.values())[i % len(TREES)]) for i in range(17)]
    seqs[3] = (700, 40)
    c = Case(ctx, "fp8", 2, 128, seqs, seed=2)
    c.fill()
    check_attention(c, 8)


def test_attention_of_a_wide_tree(ctx):
    rng = np.random.default_rng(4)
    parents = [-1] + [int(rng.integers(max(-1, i - 20), i)) for i in range(1, 150)]
    c = Case(ctx, "int8", 1, 128, [(77, parents)], seed=4)
    c.fill()
    check_attention(c, 4)


@pytest.mark.parametrize("fmt", gpu.KV_FORMATS)
def test_what_is_masked_does_not_reach_a_row(ctx, fmt):
    """NaN, infinities and the largest values in siblings' rows, and in the slots behind the sequence."""
    tree = [-1, 0, 0, 1, 2]
    c = Case(ctx, fmt, 2, 64, [(20, tree)], seed=8)
    c.fill()
    q = c.rng.standard_normal((5, 4, 64)).astype(np.float32)
    clean = check_attention(c, 4, q)
    for worst in (np.nan, np.inf, 3e38, -3e38):
        for x in (c.k, c.v):
            x[0][22] = worst      # row 2, which rows 0, 1 and 3 do not see
        c.fill()
        table = c.tables[0]
        behind = gpu.Rows(ctx, c.kv, [gpu.TreeSeq(25, table, 7)])
        junk = torch.full((7, 2, 64), float(worst), device="cuda")
        out = torch.empty(5, 4, 64, device="cuda")
        qd = cuda(q)
        torch.cuda.synchronize()
        gpu.kv_append(ctx, behind, c.kv, 0, junk, junk)
        gpu.tree_attention(ctx, c.rows(4), c.kv, 0, qd, out)
        ctx.sync()
        got = out.cpu().numpy()
        for r in (0, 1, 3):
            assert np.array_equal(got[r], clean[r]), (worst, r)


def test_peaked_scores_and_equal_ones(ctx):
    c = Case(ctx, "int8", 1, 64, [(500, 2)], seed=9)
    c.k[0][:250] = c.k[0][0]
    c.fill()
    q = c.rng.standard_normal((2, 2, 64)).astype(np.float32)
    q[0] *= 30
    q[1, 1] = 0  # every token alike
    check_attention(c, 2, q)


@pytest.mark.parametrize("fmt", ["int8", "f32"])
def test_rows_planned_again_and_outputs_apart(ctx, fmt):
    """set() with larger and smaller rows between calls in flight, strided queries and outputs, out = q."""
    c = Case(ctx, fmt, 2, 32, [(40, TREES["deep"]), (900, 3)], seed=11)
    c.fill()
    rows = gpu.Rows(ctx, c.kv, [gpu.TreeSeq(40, c.tables[0], 1)], heads=4)
    wide = [cuda(c.rng.standard_normal((13, 6, 32)).astype(np.float32)) for _ in range(2)]
    outs = []
    torch.cuda.synchronize()
    for seqs in ([gpu.TreeSeq(40, c.tables[0], TREES["deep"]), gpu.TreeSeq(900, c.tables[1], 3)],
                 [gpu.TreeSeq(900, c.tables[1], 3)], [gpu.TreeSeq(40, c.tables[0], TREES["deep"])]):
        rows.set(seqs)
        out = torch.full((13, 7, 32), 5.0, device="cuda")
        torch.cuda.synchronize()
        gpu.tree_attention(ctx, rows, c.kv, 0, wide[0][:rows.total, 1:5], out[:rows.total, 2:6])
        outs.append((rows.total, out))
    ctx.sync()
    (a, x), (b, y), (d, z) = [(n, o.cpu().numpy()) for n, o in outs]
    assert (a, b, d) == (13, 3, 10)
    for n, o in ((a, x), (b, y), (d, z)):
        assert (o[:, :2] == 5).all() and (o[:, 6:] == 5).all() and (o[n:] == 5).all()
    q = wide[0][:, 1:5].cpu().numpy()
    hk, hv = [held(k, fmt) for k in c.k], [held(v, fmt) for v in c.v]
    for got, qs, s in ((x[:10], q[:10], 0), (x[10:], q[10:], 1), (y[:3], q[:3], 1), (z[:10], q[:10], 0)):
        want, tol = attention64(qs, hk[s], hv[s], sees(c.pos[s], c.parents[s]), fmt)
        assert (np.abs(got[:, 2:6] - want) <= tol).all()
    same = wide[0][:10, 1:5].contiguous()
    torch.cuda.synchronize()
    gpu.tree_attention(ctx, rows, c.kv, 0, same, same)
    ctx.sync()
    assert np.array_equal(same.cpu().numpy(), z[:10, 2:6])
