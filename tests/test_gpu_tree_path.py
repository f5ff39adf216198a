"""The model paths over 8-bit caches and drafted trees: fg_forward and the
speculative steps on every cache format, fg_forward_tree, fg_tree_step, and
the runner that drafts trees, on the golden models.

On an 8-bit cache a forward is checked against a 64-bit forward that takes its
keys and values from the device's cache: the logits must agree to LOGIT_TOL,
as on the f32 cache, and the cached values must be the 64-bit ones to half a
quantization step plus the f32 error (1e-4 of the row's largest, LOGIT_TOL)."""
import numpy as np
import pytest

import oracle
from conftest import FIXTURES, GOLDEN, LOGIT_TOL, assert_argmax_parity
from ferrolm_amd import gpu
from ferrolm_amd.spec import Runner, TreeRunner, generate, generate_tree
from ferrolm_amd.weights import load_model

pytestmark = pytest.mark.gpu
STEP = {"int8": 0.5 / 127, "fp8": 2.0 ** -4}  # half a step, of the row's largest


def prompt(n, vocab, seed=1):
    return np.random.default_rng(seed).integers(3, vocab, n).astype(np.uint32)


def rope(c, x, pos):
    f = 1.0 / c.rope_theta ** (np.arange(0, c.head_dim, 2) / c.head_dim)
    if c.rope_llama3:
        wave = 2 * np.pi / f
        low, high = c.rope_orig_max_pos / c.rope_low_freq, c.rope_orig_max_pos / c.rope_high_freq
        smooth = (c.rope_orig_max_pos / wave - c.rope_low_freq) / (c.rope_high_freq - c.rope_low_freq)
        f = np.where(wave < high, f, np.where(wave > low, f / c.rope_factor, (1 - smooth) * f / c.rope_factor + smooth * f))
    a = np.float32(pos)[:, None] * f.astype(np.float32)[None]
    cos, sin = np.cos(a.astype(np.float64))[:, None], np.sin(a.astype(np.float64))[:, None]
    u, v = np.split(x, 2, axis=-1)
    return np.concatenate([u * cos - v * sin, v * cos + u * sin], axis=-1)


def forward64(hm, tokens, pos, visible, cached):
    """Logits of rows at positions `pos` that see visible [rows][cached tokens]; cached: per layer the (k, v)
    [tokens][kv_heads][hd] that the device holds. Returns (logits, per layer the rows' own k and v)."""
    c = hm.cfg
    x = (hm.embed.reshape(c.vocab, c.hidden).astype(np.uint32) << 16).view(np.float32).astype(np.float64)[tokens]
    own = []

    def norm(v, w):
        return v / np.sqrt((v * v).mean(1, keepdims=True) + c.rms_eps) * w

    for l, (ck, cv) in zip(hm.layers, cached):
        y = norm(x, l.attn_norm) @ l.wqkv.to_f32().astype(np.float64).T
        if l.bqkv is not None:
            y = y + l.bqkv
        q, k, v = np.split(y, [c.q_dim, c.q_dim + c.kv_heads * c.head_dim], axis=1)
        q = rope(c, q.reshape(len(x), -1, c.head_dim), pos)
        own.append((rope(c, k.reshape(len(x), -1, c.head_dim), pos), v.reshape(len(x), -1, c.head_dim)))
        o = np.zeros_like(q)
        for h in range(c.heads):
            g = h * c.kv_heads // c.heads
            s = np.where(visible, q[:, h] @ ck[:, g].T / np.sqrt(c.head_dim), -np.inf)
            w = np.exp(s - s.max(1, keepdims=True))
            o[:, h] = w / w.sum(1, keepdims=True) @ cv[:, g]
        x = x + o.reshape(len(x), -1) @ l.wo.to_f32().astype(np.float64).T
        gate, up = np.split(norm(x, l.mlp_norm) @ l.w_gate_up.to_f32().astype(np.float64).T, 2, axis=1)
        x = x + (gate / (1 + np.exp(-gate)) * up) @ l.w_down.to_f32().astype(np.float64).T
    head = hm.embed if hm.lm_head is None or c.tie_embeddings else hm.lm_head
    return norm(x, hm.norm) @ (head.reshape(c.vocab, c.hidden).astype(np.uint32) << 16).view(np.float32).astype(np.float64).T, own


def held(kv, cfg, table, n):
    """Per layer the k and v of n tokens [tokens][kv_heads][hd], in 64 bits."""
    at = np.asarray(table)[np.arange(n) // 16], np.arange(n) % 16
    out = []
    for i in range(cfg.layers):
        k, v = (a.reshape(-1, cfg.kv_heads, 16, cfg.head_dim)[at[0], :, at[1]].astype(np.float64) for a in kv.layer(i))
        out.append((k, v))
    return out


def check_cached(own, cached, fmt):
    for (k, v), (ck, cv) in zip(own, cached):
        for a, b in ((k, ck), (v, cv)):
            top = np.abs(a).max(axis=-1, keepdims=True)
            assert (np.abs(a - b) <= top * (STEP.get(fmt, 0) * 1.001 + LOGIT_TOL)).all()


@pytest.mark.parametrize("name", FIXTURES)
@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_forwards_over_an_8_bit_cache(ctx, name, fmt):
    """A prompt chunk, a second one, a decode row and verify rows, through every row count's kernels."""
    hm = load_model(GOLDEN / name)
    m = gpu.Model(ctx, hm)
    kv = gpu.KvCache(ctx, hm.cfg, 24, format=fmt)
    table = [5, 2, 9, 11, 0, 7, 21, 3, 1]
    toks = prompt(120, hm.cfg.vocab)
    at = 0
    for n in (40, 33, 1, 4, 17):
        o = gpu.forward(ctx, m, kv, [(toks[at:at + n], at, table, gpu.LOGITS_ALL)])
        cached = held(kv, hm.cfg, table, at + n)
        visible = np.arange(at + n)[None] <= (at + np.arange(n))[:, None]
        want, own = forward64(hm, toks[at:at + n], at + np.arange(n), visible, cached)
        check_cached(own, [(k[at:], v[at:]) for k, v in cached], fmt)
        assert np.abs(o.logits - want).max() <= LOGIT_TOL * np.abs(want).max()
        assert_argmax_parity(o.argmax, want)
        at += n


@pytest.mark.parametrize("name", FIXTURES)
@pytest.mark.parametrize("fmt", gpu.KV_FORMATS)
def test_forward_over_trees(ctx, name, fmt):
    hm = load_model(GOLDEN / name)
    m = gpu.Model(ctx, hm)
    kv = gpu.KvCache(ctx, hm.cfg, 40, format=fmt)
    trees = [(37, [-1, 0, 0, 1, 1, 2, 3]), (0, [-1, -1, 0, 2, 2]), (16, [-1]), (50, 21)]
    toks = [prompt(n + (p if isinstance(p, int) else len(p)), hm.cfg.vocab, s) for s, (n, p) in enumerate(trees)]
    tables = [[1, 4, 6], [9], [20, 21], [30, 31, 32, 33, 39]]
    for (n, _), t, b in zip(trees, toks, tables):
        if n:
            gpu.forward(ctx, m, kv, [(t[:n], 0, b, gpu.LOGITS_NONE)])
    o = gpu.forward_tree(ctx, m, kv, [gpu.TreeSeq(n, b, p, t[n:]) for (n, p), t, b in zip(trees, toks, tables)])
    at = 0
    for (n, p), t, b in zip(trees, toks, tables):
        p = list(range(-1, p - 1)) if isinstance(p, int) else p
        vis = np.zeros((len(p), n + len(p)), bool)
        depth = []
        for i, x in enumerate(p):
            depth.append(0 if x < 0 else depth[x] + 1)
            vis[i] = vis[x] if x >= 0 else np.arange(n + len(p)) < n
            vis[i, n + i] = True
        cached = held(kv, hm.cfg, b, n + len(p))
        want, own = forward64(hm, t[n:], n + np.array(depth), vis, cached)
        check_cached(own, [(k[n:], v[n:]) for k, v in cached], fmt)
        got = o.logits[at:at + len(p)]
        assert np.abs(got - want).max() <= LOGIT_TOL * np.abs(want).max()
        assert_argmax_parity(o.argmax[at:at + len(p)], want)
        at += len(p)


@pytest.mark.parametrize("fmt", gpu.KV_FORMATS)
@pytest.mark.parametrize("sampled", [False, True])
def test_tree_step_is_forward_walk_and_commit(ctx, fmt, sampled):
    """Against forward_tree on a second cache: the same tokens, and the branch's rows in place."""
    from test_gpu_tree_verify import walk
    hm = load_model(GOLDEN / "llama-gqa")
    c, m = hm.cfg, gpu.Model(ctx, hm)
    kvs = [gpu.KvCache(ctx, c, 40, format=fmt) for _ in range(2)]
    lengths, tables = [29, 3, 64], [[1, 4, 6], [9, 10], [20, 21, 22, 23, 24, 25]]
    parents = [-1, 0, 0, 1, 1, 2, 3, 6]
    toks = [prompt(n, c.vocab, 10 + s) for s, n in enumerate(lengths)]
    for kv in kvs:
        gpu.forward(ctx, m, kv, [(t, 0, b, gpu.LOGITS_NONE) for t, b in zip(toks, tables)])
    # drafts that pass somewhere: the target's own likeliest tokens behind each row, found level by level
    trees = [[int(prompt(1, c.vocab, 90 + s)[0])] + [0] * 7 for s in range(3)]
    for level in ([1, 2], [3, 4, 5], [6], [7]):
        o = gpu.forward_tree(ctx, m, kvs[0], [gpu.TreeSeq(n, b, parents, t) for n, b, t in zip(lengths, tables, trees)])
        for s in range(3):
            for i in level:
                kids = [x for x in range(8) if parents[x] == parents[i]]
                trees[s][i] = int(np.argsort(-o.logits[8 * s + parents[i]], kind="stable")[kids.index(i) + (s == 1)])
    seqs = [gpu.TreeSeq(n, b, parents, t) for n, b, t in zip(lengths, tables, trees)]
    o = gpu.forward_tree(ctx, m, kvs[0], seqs)
    params = u = None
    if sampled:
        params = [gpu.SamplingParams(0.8, 0.95, 0), gpu.SamplingParams(1.0, 1.0, 40), gpu.SamplingParams(0.0)]
        u = np.random.default_rng(5).random(24, np.float32)
    out, path = gpu.tree_step(ctx, m, kvs[1], seqs, params, u)
    for s in range(3):
        r = slice(8 * s, 8 * s + 8)
        if sampled and s < 2:
            p = np.zeros((8, c.vocab), np.float32)
            for i in range(8):
                ids, pr = oracle.distribution(o.logits[8 * s + i], params[s].temperature, params[s].top_p, params[s].top_k)
                p[i, np.asarray(ids)] = pr
            want, way = walk(parents, trees[s], p, None, u[r], "fixed")
        else:
            node, want, way = 0, [], []
            while node is not None:
                way.append(node)
                want.append(int(o.argmax[8 * s + node]))
                node = next((i for i in range(8) if parents[i] == node and trees[s][i] == want[-1]), None)
        assert out[s].tolist() == want and path[s].tolist() == way
        a, b = held(kvs[0], c, tables[s], lengths[s] + 8), held(kvs[1], c, tables[s], lengths[s] + 8)
        for (ak, av), (bk, bv) in zip(a, b):
            for x, y in ((ak, bk), (av, bv)):
                w = x.copy()
                for j, row in enumerate(way):
                    w[lengths[s] + j] = x[lengths[s] + row]
                assert np.array_equal(w, y)


@pytest.mark.parametrize("name", FIXTURES)
def test_tree_generation_is_the_greedy_one(ctx, name):
    hm = load_model(GOLDEN / name)
    m = gpu.Model(ctx, hm)
    draft = m.truncated(1)
    p = prompt(45, hm.cfg.vocab)
    om = oracle.Model(hm)
    want, _, _ = oracle.generate(om, om.truncated(1), [int(t) for t in p], 40, 3, kv_blocks=64)
    for fans in ((4, 2, 1), (1, 1, 1), (2,), (3, 3)):
        got = generate_tree(ctx, m, draft, p, 40, fans, kv_blocks=64, max_batch_tokens=20)
        assert np.array_equal(got, want), fans


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_generation_over_8_bit_caches(ctx, fmt):
    """Chains, trees and plain steps over one format. Their rows go through products of other row counts,
    which may round a key to another code: tokens may part where two logits are as near as that, so each
    generation's own tokens are checked against the logits of a fresh forward over them, to half a step of
    one code in 32 channels of a row (its share of a score) and LOGIT_TOL."""
    hm = load_model(GOLDEN / "llama-gqa")
    c, m = hm.cfg, gpu.Model(ctx, hm)
    draft = m.truncated(1)
    p = [int(t) for t in prompt(50, c.vocab, 3)]

    def cache(model):
        return gpu.KvCache(ctx, model.cfg, 64, format=fmt)

    runs = [generate(ctx, m, draft, p, 32, 3, kv_blocks=64, tkv=cache(m), dkv=cache(draft), max_seqs=0),
            generate(ctx, m, None, p, 32, 0, kv_blocks=64, tkv=cache(m)),
            generate_tree(ctx, m, draft, p, 32, (3, 2, 1), kv_blocks=64, kv_format=fmt)]
    for got in runs:
        assert len(got) == 32
        whole = p + [int(t) for t in got]
        o = gpu.forward(ctx, m, cache(m), [(whole[:-1], 0, list(range(8)), gpu.LOGITS_ALL)])
        lg = o.logits[len(p) - 1:]
        gap = lg.max(1) - lg[np.arange(32), got]
        assert (gap <= (STEP[fmt] / 32 + 2 * LOGIT_TOL) * np.abs(lg).max(1)).all(), gap


def test_sampled_tree_generation_runs_on_its_seed(ctx):
    hm = load_model(GOLDEN / "llama-gqa")
    m = gpu.Model(ctx, hm)
    draft = m.truncated(1)
    p = prompt(20, hm.cfg.vocab)
    runs = [generate_tree(ctx, m, draft, p, 24, (3, 2), kv_blocks=16, kv_format="int8",
                          params=gpu.SamplingParams(0.9, 0.95, 50, seed)) for seed in (1, 1, 2)]
    assert np.array_equal(runs[0], runs[1]) and not np.array_equal(runs[0], runs[2])
    assert all(len(r) == 24 and (r < hm.cfg.vocab).all() for r in runs)


def test_a_tree_run_ends_at_the_context_limit(ctx):
    hm = load_model(GOLDEN / "llama-gqa")
    m = gpu.Model(ctx, hm)
    r = generate_tree(ctx, m, m.truncated(1), prompt(20, hm.cfg.vocab), 500, (2, 2), kv_blocks=4)
    assert len(r) == 4 * 16 - 20


def shaped(kind, hidden, heads, kv_heads, hd, inter, seed, bias=False):
    from ferrolm_amd import synth
    from ferrolm_amd.weights import Config
    c = Config(vocab=608, hidden=hidden, intermediate=inter, layers=2, heads=heads, kv_heads=kv_heads, head_dim=hd,
               rms_eps=1e-5, rope_theta=1e4, max_position=1024, tie_embeddings=True, qkv_bias=bias, eos=(0,))
    return synth.quantize_model(synth.random_model(c, seed), kind)


@pytest.mark.parametrize("fmt", gpu.KV_FORMATS)
@pytest.mark.parametrize("kind,shape", [(0, (576, 9, 3, 64, 1536)), (2, (1024, 16, 16, 64, 2048)),
                                        (1, (1024, 16, 2, 128, 1024)), (0, (256, 8, 1, 32, 512))])
def test_wide_models_over_every_cache(ctx, fmt, kind, shape):
    """Head dims and weight kinds of the served models, through the fused small steps, the GEMVs and the GEMMs:
    prompt, decode rows of several sequences, trees."""
    hm = shaped(kind, *shape, seed=shape[0])
    c, m = hm.cfg, gpu.Model(ctx, hm)
    kv = gpu.KvCache(ctx, c, 64, format=fmt)
    tables = [[3 * i + s for i in range(12)] for s in range(3)]
    toks = [prompt(150, c.vocab, 40 + s) for s in range(3)]
    at = [0, 0, 0]

    def check(rows, call):
        """rows: per sequence the parents of its rows"""
        o = call([toks[s][at[s]:at[s] + len(rows[s])] for s in range(3)])
        i = 0
        for s in range(3):
            n, p = at[s], rows[s]
            vis, depth = np.zeros((len(p), n + len(p)), bool), []
            for j, x in enumerate(p):
                depth.append(0 if x < 0 else depth[x] + 1)
                vis[j] = vis[x] if x >= 0 else np.arange(n + len(p)) < n
                vis[j, n + j] = True
            want, own = forward64(hm, toks[s][n:n + len(p)], n + np.array(depth), vis, held(kv, c, tables[s], n + len(p)))
            check_cached(own, [(k[n:], v[n:]) for k, v in held(kv, c, tables[s], n + len(p))], fmt)
            got = o.logits[i:i + len(p)]
            assert np.abs(got - want).max() <= LOGIT_TOL * np.abs(want).max()
            i += len(p)
    for n in ((70, 33, 9), (1, 1, 1), (2, 1, 1), (3, 5, 12)):
        check([list(range(-1, k - 1)) for k in n],
              lambda t: gpu.forward(ctx, m, kv, [(t[s], at[s], tables[s], gpu.LOGITS_ALL) for s in range(3)]))
        at = [a + k for a, k in zip(at, n)]
    trees = [[-1, 0, 0, 1], [-1, -1, 0, 1, 1, 2, 2, 6], [-1]]
    check(trees, lambda t: gpu.forward_tree(ctx, m, kv, [gpu.TreeSeq(at[s], tables[s], trees[s], t[s]) for s in range(3)]))


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_speculative_steps_on_8_bit_caches_with_and_without_graphs(ctx, fmt, monkeypatch):
    """The same launches captured and direct: the same tokens, over enough steps that contexts pass block and
    plan boundaries."""
    hm = shaped(0, 576, 9, 3, 64, 1536, seed=5)
    outs = []
    for no_graph in ("0", "1"):
        monkeypatch.setenv("FERRO_NO_GRAPH", no_graph)
        x = gpu.Context(0)
        m = gpu.Model(x, hm)
        d = m.truncated(1)
        p = prompt(30, hm.cfg.vocab)
        outs.append(generate(x, m, d, p, 120, 3, kv_blocks=32, tkv=gpu.KvCache(x, hm.cfg, 32, format=fmt),
                             dkv=gpu.KvCache(x, d.cfg, 96, format=fmt)))
    assert np.array_equal(outs[0], outs[1])


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_capture_on_an_8_bit_cache(ctx, fmt):
    """The first layer's attention rows of a calibration capture: over what the cache holds."""
    hm = load_model(GOLDEN / "llama-gqa")
    c, m, p = hm.cfg, gpu.Model(ctx, hm), prompt(37, hm.cfg.vocab)
    kv = gpu.KvCache(ctx, c, 8, format=fmt)
    x, got = gpu.forward_capture(ctx, m, kv, [(p, 0, [4, 1, 2])])[0][:2]
    (ck, cv), n, l = held(kv, c, [4, 1, 2], 37)[0], 37, hm.layers[0]
    q = (x.astype(np.float64) @ l.wqkv.to_f32().astype(np.float64).T + (0 if l.bqkv is None else l.bqkv))[:, :c.q_dim]
    q = rope(c, q.reshape(n, -1, c.head_dim), np.arange(n))
    want = np.zeros_like(q)
    for h in range(c.heads):
        g = h * c.kv_heads // c.heads
        s = np.where(np.tri(n, dtype=bool), q[:, h] @ ck[:, g].T / np.sqrt(c.head_dim), -np.inf)
        w = np.exp(s - s.max(1, keepdims=True))
        want[:, h] = w / w.sum(1, keepdims=True) @ cv[:, g]
    assert np.abs(got - want.reshape(n, -1)).max() <= LOGIT_TOL * np.abs(want).max()


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("spec_k", [0, 3])
def test_the_engine_serves_from_8_bit_caches(ctx, fmt, spec_k):
    """Requests of a shared prefix, chunked and overlapping, plain and speculative: each one's tokens against the
    logits of a fresh forward over them, as the generations above."""
    from ferrolm_amd.engine import Engine, EngineConfig, Params
    hm = load_model(GOLDEN / "llama-gqa")
    c, m = hm.cfg, gpu.Model(ctx, hm)
    e = Engine(ctx, m, m.truncated(1) if spec_k else None,
               EngineConfig(kv_blocks=64, kv_format=fmt, spec_k=spec_k or 4, max_batch_tokens=40, max_seqs=2))
    assert e.kv.format == fmt and (not spec_k or e.dkv.format == fmt)
    first = [int(t) for t in prompt(40, c.vocab, 9)]
    prompts = [first + [int(t) for t in prompt(3 + 9 * i, c.vocab, i)] for i in range(4)]
    reqs = [e.submit(p, Params(max_tokens=12, ignore_eos=True)) for p in prompts]
    e.run_until_idle()
    for p, r in zip(prompts, reqs):
        assert len(r.tokens) == 12
        whole = p + [int(t) for t in r.tokens]
        o = gpu.forward(ctx, m, gpu.KvCache(ctx, c, 8, format=fmt), [(whole[:-1], 0, list(range(8)), gpu.LOGITS_ALL)])
        lg = o.logits[len(p) - 1:]
        assert (lg.max(1) - lg[np.arange(12), r.tokens] <= (STEP[fmt] / 32 + 2 * LOGIT_TOL) * np.abs(lg).max(1)).all()
