"""The operators of tree speculation over an 8-bit paged cache, as a serving program calls them.

A verify step of drafted token trees runs, in every layer, a cache write
(`store`: keys and values quantized row by row as they enter the pages, and
read back) and an attention of the tree's rows over the cached context
(`attend`), and after the last layer one walk down the tree against the
target's distributions (`verify`). A whole context is read back when a prefix
moves to another cache (`gather`).

Where `own` is false, `run` computes them in plain torch; where it is true, it
calls ferrolm_amd.gpu.

Quantization (bit for bit, in 32-bit steps): a row of one head has the scale
s = max|x| / 127 (int8) or / 448 (fp8 e4m3), its codes are x / s rounded to
nearest, ties to even, and stand for code * s.

Attention of row i of a sequence whose cached context is `pos` tokens: over
all of them and over the rows of its own branch, itself included; a chain's
row sees every row before it.

Verification: at a node with target distribution p and draft distribution q,
the children are tried in order; child c passes when u * q(c) < P(c), P being
p after the rejections so far, each of which leaves max(0, P - q) / sum
("each": children drawn independently; "distinct": without replacement, q then
without the tokens before, over its sum; "fixed": given tokens, q(c) = 1, a
rejected token's mass removed). The walk ends with a draw from what is left at
the last node: the first token whose cumulative mass exceeds u times the sum.
"""
from __future__ import annotations

import math
import zlib

import numpy as np
import torch

own = False

# (query heads, kv heads, head dim, vocabulary) of the shapes in ferrolm_amd.weights
SHAPES = {"135m": (9, 3, 64, 49152), "360m": (15, 5, 64, 49152), "1.7b": (32, 32, 64, 49152),
          "1b": (32, 8, 64, 128256), "8b": (32, 8, 128, 128256)}
LEVELS = {"int8": 127.0, "fp8": 448.0}


def listed():
    return [
        # One new token of a lone stream, and the ragged prompt chunks of a batch, into the cache and back.
        dict(name="store_token_int8", op="store", shape="8b", format="int8", seqs=1, lo=1030, hi=1030, tree="1"),
        dict(name="store_prompts_fp8", op="store", shape="8b", format="fp8", seqs=6, lo=0, hi=777, tree="chain 1900"),
        # Contexts read back in f32: two short odd ones, a batch's.
        dict(name="gather_short_fp8", op="gather", shape="135m", format="fp8", seqs=2, lo=37, hi=301, tree="1"),
        dict(name="gather_batch_int8", op="gather", shape="1.7b", format="int8", seqs=16, lo=128, hi=2048, tree="1"),
        # A plain decode step over an 8-bit cache: one token of one stream. Latency-bound.
        dict(name="attend_token_int8", op="attend", shape="1.7b", format="int8", seqs=1, lo=1030, hi=1030, tree="1"),
        # A drafted tree of one stream over the f32 cache that a server has by default.
        dict(name="attend_tree_f32", op="attend", shape="1.7b", format="f32", seqs=1, lo=1030, hi=1030, tree="4.2.1"),
        # Trees of a full batch with ragged contexts, grouped-query heads at head dim 128.
        dict(name="attend_trees_int8_b16", op="attend", shape="8b", format="int8", seqs=16, lo=512, hi=4001,
             tree="3.2.1.1"),
        # A tree at the end of a very long context: the case that an 8-bit cache is for.
        dict(name="attend_long_fp8", op="attend", shape="8b", format="fp8", seqs=1, lo=131069, hi=131069, tree="4.2.2"),
        # Prompt chunks over what is cached already: bound by the products.
        dict(name="attend_prompts_int8", op="attend", shape="8b", format="int8", seqs=2, lo=700, hi=1500,
             tree="chain 2047"),
        # Verification: one stream's tree of the draft's likeliest tokens, a batch of trees of independent draws, a
        # few bushy trees of draws without replacement.
        dict(name="verify_fixed_b1", op="verify", vocab=49152, draft="fixed", seqs=1, tree="4.2.1"),
        dict(name="verify_each_b16", op="verify", vocab=128256, draft="each", seqs=16, tree="3.2.1.1"),
        dict(name="verify_distinct_b4", op="verify", vocab=128256, draft="distinct", seqs=4, tree="8.4.2"),
    ]


def draw(rng):
    def size(lo, hi):
        """Log-uniform in [lo, hi]."""
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(("store", "gather", "attend", "attend", "attend", "verify", "verify"))
    seqs = size(1, 24)
    trees = ("1", "1", "chain %d" % rng.randint(2, 9), "2.1", "4.2.1", "3.2.1.1", "2.2.2.2", "5.1.1", "4.4")
    if op == "verify":
        return dict(op=op, vocab=rng.choice((size(2000, 40000), 49152, 128256)),
                    draft=rng.choice(("fixed", "each", "distinct")), seqs=min(seqs, 12),
                    tree=rng.choice(trees[2:] + ("6.3.1",)))
    shape = rng.choice(("135m", "360m", "1.7b", "1b", "8b"))
    lo = size(1, 40000 // seqs)
    case = dict(op=op, shape=shape, format=rng.choice(("int8", "fp8", "int8", "fp8", "f32")), seqs=seqs, lo=lo,
                hi=rng.randint(lo, min(2 * lo + 16, 48000 // seqs)), tree=rng.choice(trees))
    if op == "store" or (op == "attend" and rng.random() < 0.2):
        case |= dict(seqs=min(seqs, 4), tree="chain %d" % size(10, 1500))
        case |= dict(lo=min(case["lo"], 2000), hi=min(case["hi"], 4000))
    if op == "gather":
        case |= dict(lo=min(lo, 20000 // seqs), hi=min(case["hi"], 24000 // seqs))
    return case


# ---------------------------------------------------------------------------
# What a case consists of
# ---------------------------------------------------------------------------
def _parents(tree, s):
    """The parents of the rows of sequence s: -1 for the first row, which is the last token that is settled. Every
    second sequence's tree is a level shorter, its chain by a third."""
    if tree == "1":
        return [-1]
    if tree.startswith("chain "):
        n = int(tree[6:])
        return list(range(-1, (n if s % 2 == 0 else max(1, 2 * n // 3)) - 1))
    fans = [int(f) for f in tree.split(".")]
    parents, level = [-1], [0]
    for f in fans[:-1] if s % 2 else fans:
        first = len(parents)
        parents += [at for at in level for _ in range(f)]
        level = list(range(first, len(parents)))
    return parents


def _lengths(case):
    """The context lengths: spread evenly over [lo, hi]."""
    n, lo, hi = case["seqs"], case["lo"], max(case["lo"], case["hi"])
    return [lo + (hi - lo) * i // max(1, n - 1) for i in range(n)]


def _sequences(case):
    """(context length, parents of the new rows) of each sequence."""
    lengths = _lengths(case) if "lo" in case else [0] * case["seqs"]
    return [(n, _parents(case["tree"], s)) for s, n in enumerate(lengths)]


def _rand(seed, *key):
    g = torch.Generator("cuda")
    g.manual_seed(zlib.crc32(repr((int(seed), key)).encode()))
    return g


def _tables(seqs, seed):
    """Block tables out of a shuffled pool, as a server's pool is after some requests, and the pool's size."""
    need = [(n + len(p) + 15) // 16 for n, p in seqs]
    order = np.random.default_rng((int(seed), 7)).permutation(sum(need)).astype(np.uint32)
    ends = np.cumsum(need)
    return [order[e - n:e] for e, n in zip(ends, need)], sum(need)


def _slots(table, first, last):
    """Cache slots (block * 16 + offset) of the positions first..last-1."""
    at = np.arange(first, last)
    return table[at // 16].astype(np.int64) * 16 + at % 16


def _keys_values(tokens, kv_heads, hd, seed, what):
    """Keys or values [tokens][kv heads][head dim] as trained models have them: some channels larger, some tokens."""
    g = _rand(seed, what)
    x = torch.randn(tokens, kv_heads, hd, generator=g, device="cuda")
    x *= torch.exp(0.5 * torch.randn(1, kv_heads, hd, generator=g, device="cuda"))
    return x.mul_(torch.exp(0.3 * torch.randn(tokens, kv_heads, 1, generator=g, device="cuda")))


def _quantized(x, fmt):
    """(codes as the numbers they are, scales) of rows along the last axis, in the steps of the definition."""
    if fmt == "f32":
        return x, torch.ones_like(x[..., :1])
    s = x.abs().amax(dim=-1, keepdim=True) / LEVELS[fmt]
    c = torch.where(s > 0, x / s, torch.zeros_like(x))
    if fmt == "int8":
        return c.round().clamp_(-127, 127).to(torch.int8), s
    return c.to(torch.float8_e4m3fn), s


# ---------------------------------------------------------------------------
# The cases
# ---------------------------------------------------------------------------
_ctx = None


def _context():
    global _ctx
    if _ctx is None:
        from ferrolm_amd import gpu
        _ctx = gpu.Context(0)
    return _ctx


def _distributions(case, seqs, seed):
    """Target and draft distributions of every node: peaked as a language model's, the draft's near the target's."""
    rows = sum(len(p) for _, p in seqs)
    g = _rand(seed, "logits")
    z = torch.randn(rows, case["vocab"], generator=g, device="cuda").mul_(3.0)
    p = torch.softmax(z, dim=1)
    z += torch.randn(rows, case["vocab"], generator=g, device="cuda")
    return p, torch.softmax(z, dim=1)


def _children(seqs):
    """[rows][most children] row of each node's children in order, -1 past them; the first row of each sequence."""
    found, roots = [], []
    for _, parents in seqs:
        roots.append(len(found))
        found += [[] for _ in parents]
        for i, p in enumerate(parents):
            if p >= 0:
                found[roots[-1] + p].append(roots[-1] + i)
    most = max(1, max(len(c) for c in found))
    return np.array([c + [-1] * (most - len(c)) for c in found], np.int64), np.array(roots, np.int64)


def _drafted(case, children, q, seed):
    """A token for every row: children drawn from their parent's draft distribution, or its likeliest tokens."""
    tokens = torch.randint(0, case["vocab"], (len(children),), generator=_rand(seed, "roots"), device="cuda")
    counts = (children >= 0).sum(1)
    for n in sorted(set(counts[counts > 0].tolist())):
        nodes = np.nonzero(counts == n)[0]
        at = torch.from_numpy(nodes).cuda()
        kids = torch.from_numpy(children[nodes, :n]).cuda()
        if case["draft"] == "fixed":
            tokens[kids] = q[at].topk(n, dim=1).indices
        else:
            tokens[kids] = torch.multinomial(q[at], n, replacement=case["draft"] == "each", generator=_rand(seed, n))
    return tokens.to(torch.int32)


def _verify_inputs(case, seed):
    seqs = _sequences(case)
    p, q = _distributions(case, seqs, seed)
    children, roots = _children(seqs)
    tokens = _drafted(case, children, q, seed)
    u = torch.rand(len(children), generator=_rand(seed, "uniform"), device="cuda")
    return seqs, p, None if case["draft"] == "fixed" else q, children, roots, tokens, u


def _depth(parents):
    """Rows on the longest path of a tree."""
    depth = []
    for p in parents:
        depth.append(1 if p < 0 else depth[p] + 1)
    return max(depth)


def _attend_inputs(case, seed):
    heads, kv_heads, hd, _ = SHAPES[case["shape"]]
    seqs = _sequences(case)
    tables, blocks = _tables(seqs, seed)
    total = sum(n + len(p) for n, p in seqs)
    k = _keys_values(total, kv_heads, hd, seed, "keys")
    v = _keys_values(total, kv_heads, hd, seed, "values")
    slots = torch.from_numpy(np.concatenate([_slots(t, 0, n + len(p)) for t, (n, p) in zip(tables, seqs)])).cuda()
    return seqs, tables, blocks, k, v, slots


def _queries(case, seqs, seed):
    heads, _, hd, _ = SHAPES[case["shape"]]
    rows = sum(len(p) for _, p in seqs)
    return torch.randn(rows, heads, hd, generator=_rand(seed, "queries"), device="cuda")


def _sees(seqs):
    """[seqs][most rows][longest context and rows]: what each row attends to."""
    rows, longest = max(len(p) for _, p in seqs), max(n + len(p) for n, p in seqs)
    sees = torch.zeros(len(seqs), rows, longest, dtype=torch.bool, device="cuda")
    for s, (n, parents) in enumerate(seqs):
        new = np.tri(len(parents), dtype=bool)
        if parents != list(range(-1, len(parents) - 1)):
            new[:] = False
            for i, p in enumerate(parents):
                if p >= 0:
                    new[i] = new[p]
                new[i, i] = True
        sees[s, :len(parents), :n] = True
        sees[s, :len(parents), n:n + len(parents)] = torch.from_numpy(new).cuda()
    return sees


def _padded(counts, most):
    """[len(counts)][most]: running index of each sequence's items, 0 past them; and which are items."""
    first = np.cumsum([0] + counts[:-1])
    at = np.arange(most)[None, :]
    real = at < np.array(counts)[:, None]
    return np.where(real, first[:, None] + at, 0), real


def prepare(case, seed):
    op = case["op"]
    if op == "verify":
        seqs, p, q, children, roots, tokens, u = _verify_inputs(case, seed)
        depth = max(_depth(parents) for _, parents in seqs)
        state = dict(op=op, draft=case["draft"], p=p, q=q, tokens=tokens, u=u, depth=depth,
                     children=torch.from_numpy(children).cuda(), roots=torch.from_numpy(roots).cuda())
        if own:
            from ferrolm_amd import gpu
            state["rows"] = gpu.Rows(_context(), None, [gpu.TreeSeq(0, None, parents) for _, parents in seqs])
            state["out"] = (torch.zeros(len(seqs), depth, dtype=torch.int32, device="cuda"),
                            torch.zeros(len(seqs), depth, dtype=torch.int32, device="cuda"),
                            torch.zeros(len(seqs), dtype=torch.int32, device="cuda"))
        torch.cuda.synchronize()
        return state
    heads, kv_heads, hd, _ = SHAPES[case["shape"]]
    fmt = case["format"]
    seqs, tables, blocks, k, v, slots = _attend_inputs(case, seed)
    counts = [len(p) for _, p in seqs]
    state = dict(op=op, fmt=fmt, slots=slots, heads=heads, kv_heads=kv_heads, hd=hd)
    ends = np.cumsum([n + len(p) for n, p in seqs])
    new = np.concatenate([np.arange(e - c, e) for e, c in zip(ends, counts)])
    if op == "store":
        # the new rows as the q/k/v projection leaves them: columns of one matrix
        qkv = torch.empty(len(new), heads + 2 * kv_heads, hd, device="cuda")
        at = torch.from_numpy(new).cuda()
        qkv[:, :heads] = 0.5
        qkv[:, heads:heads + kv_heads] = k[at]
        qkv[:, heads + kv_heads:] = v[at]
        state |= dict(k=qkv[:, heads:heads + kv_heads], v=qkv[:, heads + kv_heads:], new=slots[at])
    if op == "attend":
        index, real = _padded(counts, max(counts))
        state |= dict(q=_queries(case, seqs, seed), sees=_sees(seqs), real=torch.from_numpy(real).cuda(),
                      index=torch.from_numpy(index).cuda())
        index, _ = _padded([n + len(p) for n, p in seqs], max(n + len(p) for n, p in seqs))
        state["context"] = slots[torch.from_numpy(index).cuda()]
    if own:
        from ferrolm_amd import gpu
        state["kv"] = kv = gpu.KvCache(_context(), gpu.CacheShape(1, kv_heads, hd), blocks, format=fmt)
        state["rows"] = gpu.Rows(_context(), kv, [gpu.TreeSeq(n, t, p) for t, (n, p) in zip(tables, seqs)], heads=heads)
        whole = gpu.Rows(_context(), kv, [gpu.TreeSeq(0, t, n + len(p)) for t, (n, p) in zip(tables, seqs)])
        torch.cuda.synchronize()  # the keys and values come from another stream
        gpu.kv_append(_context(), whole, kv, 0, k, v)
        rows = len(slots) if op == "gather" else len(new)
        state["out"] = (torch.empty(rows, kv_heads, hd, device="cuda"), torch.empty(rows, kv_heads, hd, device="cuda"))
        if op == "attend":
            state["out"] = torch.empty(rows, heads, hd, device="cuda")
        _context().sync()
    else:
        (kc, ks), (vc, vs) = _quantized(k, fmt), _quantized(v, fmt)
        for name, x in (("kc", kc), ("ks", ks), ("vc", vc), ("vs", vs)):
            pool = torch.zeros(blocks * 16, *x.shape[1:], dtype=x.dtype, device="cuda")
            pool.view(torch.uint8)[slots] = x.contiguous().view(torch.uint8)
            state[name] = pool
    torch.cuda.synchronize()
    return state


def _read(state, which, slots):
    """The cached keys ("k") or values ("v") of some slots, in f32."""
    codes = state[which + "c"]
    x = codes.view(torch.int8)[slots].view(codes.dtype) if codes.dtype == torch.float8_e4m3fn else codes[slots]
    return x.float() * state[which + "s"][slots]


def _write(state, which, slots, x):
    codes, s = _quantized(x, state["fmt"])
    pool = state[which + "c"]
    if pool.dtype == torch.float8_e4m3fn:
        pool, codes = pool.view(torch.int8), codes.view(torch.int8)
    pool[slots] = codes
    state[which + "s"][slots] = s


def _attend(state):
    q, sees = state["q"], state["sees"]
    n, hd = sees.shape[1], state["hd"]
    seqs, kv_heads, group = len(sees), state["kv_heads"], state["heads"] // state["kv_heads"]
    k = _read(state, "k", state["context"]).transpose(1, 2)  # [seqs][kv heads][context][hd]
    v = _read(state, "v", state["context"]).transpose(1, 2)
    x = q[state["index"]].reshape(seqs, n, kv_heads, group, hd).permute(0, 2, 3, 1, 4).reshape(seqs, kv_heads, -1, hd)
    w = (x @ k.transpose(2, 3)).div_(math.sqrt(hd)).view(seqs, kv_heads, group, n, -1)
    w.masked_fill_(~sees[:, None, None], -math.inf)
    w -= w.amax(dim=-1, keepdim=True).clamp_min_(torch.finfo(torch.float32).min)
    w.exp_()
    total = w.sum(dim=-1, keepdim=True)
    out = (w.view(seqs, kv_heads, group * n, -1) @ v).view(seqs, kv_heads, group, n, hd) / total
    return out.permute(0, 3, 1, 2, 4).reshape(seqs, n, state["heads"], hd)[state["real"]]


def _verify(state):
    p, q, tokens, u, children, roots = (state[n] for n in ("p", "q", "tokens", "u", "children", "roots"))
    u, seqs, draft = u.double(), len(roots), state["draft"]
    tokens = tokens.long()
    out = torch.zeros(seqs, state["depth"], dtype=torch.int32, device="cuda")
    path = torch.full_like(out, -1)
    path[:, 0] = 0
    node, count = roots.clone(), torch.ones_like(roots)
    going = torch.ones(seqs, dtype=torch.bool, device="cuda")
    left = p[node].double()  # unnormalised; `total` is its sum
    total = torch.ones(seqs, 1, dtype=torch.float64, device="cuda")
    every = torch.arange(seqs, device="cuda")
    for level in range(1, state["depth"]):
        passed = torch.zeros_like(going)
        drafted = q[node].double() if q is not None else None
        here = children[node]
        for j in range(children.shape[1]):
            child = here[:, j]
            open_ = going & ~passed & (child >= 0)
            c = tokens[child.clamp_min(0)][:, None]
            mass = left.gather(1, c) / total
            rate = drafted.gather(1, c) if q is not None else torch.ones_like(mass)
            good = open_ & ((u[child.clamp_min(0)][:, None] * rate < mass) & (rate > 0))[:, 0]
            lost = (open_ & ~good)[:, None]
            if q is None:
                rest = left.scatter(1, c, 0.0)
                left, total = torch.where(lost, rest, left), torch.where(lost, total - mass * total, total)
            else:
                rest = (left / total - drafted).clamp_min_(0.0)
                left = torch.where(lost, rest, left)
                total = torch.where(lost, rest.sum(dim=1, keepdim=True), total)
                if draft == "distinct":
                    drafted = torch.where(lost, drafted.scatter(1, c, 0.0) / (1.0 - rate), drafted)
            rows = every[good]
            node[rows] = child[rows]
            out[rows, level - 1] = tokens[child[rows]].int()
            path[rows, level] = (child - roots)[rows].int()
            left[rows] = p[node[rows]].double()
            total[rows] = 1.0
            passed |= good
        going &= passed
        count += going
    left = torch.where((left.sum(dim=1, keepdim=True) > 0), left, p[node].double())
    cumulative = left.cumsum(dim=1)
    drawn = (cumulative <= u[roots][:, None] * cumulative[:, -1:]).sum(dim=1)
    last = (left > 0).long().cumsum(dim=1).argmax(dim=1)
    out[every, count - 1] = torch.minimum(drawn, last).int()
    return out, path, count.int()


def run(state):
    op = state["op"]
    if own:
        from ferrolm_amd import gpu
        ctx, rows, out = _ctx, state["rows"], state["out"]
        if op == "verify":
            gpu.tree_verify(ctx, rows, state["tokens"], state["p"], state["q"], state["u"], state["draft"], *out)
        elif op == "attend":
            gpu.tree_attention(ctx, rows, state["kv"], 0, state["q"], out)
        elif op == "store":
            gpu.kv_append(ctx, rows, state["kv"], 0, state["k"], state["v"])
            gpu.kv_gather(ctx, rows, state["kv"], 0, *out, context=False)
        else:
            gpu.kv_gather(ctx, rows, state["kv"], 0, *out)
        return out
    if op == "verify":
        return _verify(state)
    if op == "attend":
        return _attend(state)
    if op == "store":
        _write(state, "k", state["new"], state["k"])
        _write(state, "v", state["new"], state["v"])
        return _read(state, "k", state["new"]), _read(state, "v", state["new"])
    return _read(state, "k", state["slots"]), _read(state, "v", state["slots"])


def work(case):
    seqs = _sequences(case)
    rows = sum(len(p) for _, p in seqs)
    if case["op"] == "verify":
        # the distributions of each sequence's last node
        return dict(bytes=len(seqs) * case["vocab"] * (4.0 if case["draft"] == "fixed" else 8.0), flops=0.0)
    heads, kv_heads, hd, _ = SHAPES[case["shape"]]
    held = 2.0 * kv_heads * (4 * hd if case["format"] == "f32" else hd + 4)  # bytes of a token's keys and values
    whole = 8.0 * kv_heads * hd  # in f32
    if case["op"] == "store":
        return dict(bytes=rows * (2 * whole + 2 * held), flops=0.0)
    tokens = sum(n + len(p) for n, p in seqs)
    if case["op"] == "gather":
        return dict(bytes=tokens * (held + whole), flops=0.0)
    pairs = 0
    for n, parents in seqs:
        depth = []
        for p in parents:
            depth.append(1 if p < 0 else depth[p] + 1)
        pairs += n * len(parents) + sum(depth)
    return dict(bytes=tokens * held + 8.0 * rows * heads * hd, flops=4.0 * hd * heads * pairs)


# ---------------------------------------------------------------------------
# The same in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    if case["op"] in ("store", "verify"):
        return None  # defined bit for bit in 32-bit steps; whole numbers
    seqs, tables, blocks, k, v, slots = _attend_inputs(case, seed)
    # what the cache holds is the operators' input
    k, v = ((c.double() * s.double()) for c, s in (_quantized(x, case["format"]) for x in (k, v)))
    if case["op"] == "gather":
        return k, v
    heads, kv_heads, hd, _ = SHAPES[case["shape"]]
    q = _queries(case, seqs, seed).double()
    out, row, first = torch.empty_like(q), 0, 0
    for n, parents in seqs:
        branch = []  # of each row: the rows that it sees
        for i, p in enumerate(parents):
            branch.append((branch[p] if p >= 0 else []) + [i])
        hidden = torch.ones(len(parents), n + len(parents), dtype=torch.bool)
        hidden[:, :n] = False
        for i, b in enumerate(branch):
            hidden[i, [n + j for j in b]] = False
        hidden = hidden.cuda()
        last = first + n + len(parents)
        for h in range(heads):
            kh, vh = k[first:last, h * kv_heads // heads], v[first:last, h * kv_heads // heads]
            score = (q[row:row + len(parents), h] @ kh.T * hd ** -0.5).masked_fill(hidden, -math.inf)
            out[row:row + len(parents), h] = torch.softmax(score, dim=1) @ vh
        row, first = row + len(parents), last
    return out
