"""The 8-bit cache and drafted trees inside the framework: the attention mixer over an 8-bit cache against its formula on the
rows that the cache gives back, models stepped with 8-bit caches (poisoned and not) and with trees whose every token must
get the logits of its own path, generation with and without graphs."""

import random

import numpy as np
import pytest
import torch

import helpers as H
import plain_model as P

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
DT = {"float32": torch.float32, "bfloat16": torch.bfloat16}
KINDS = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
# Logits against the float32 plain implementation.  A cache in the compute type: as the replay tests bound them (inputs of
# the products and the cache rounded to bfloat16, an element off by at most 2^-9 of itself at its magnitude's middle).
TOL = {"float32": {"A": 1e-5, "B": 1e-5, "C": 1e-5, "D": 1e-5, "E": 5e-5},
       "bfloat16": {"A": 8e-3, "B": 1.2e-2, "C": 1.2e-2, "D": 1.2e-2, "E": 6e-1}}
# Codes: an element is off by at most max / 254 in int8 (a row's maximum is three to four standard deviations: 1.6 % of one),
# by 2^-4 of itself in e4m3, where bfloat16 has 2^-8: 4 and 16 times bfloat16's, whose bounds are scaled by that.
CODES = {"int8": 4, "e4m3": 16}


def tol(name, dtype, kv="auto"):
    return TOL[dtype][name] if kv == "auto" else CODES[kv] * TOL["bfloat16"][name]


@pytest.fixture(scope="module", params=["A", "B", "C", "D", "E"])
def model(request, tmp_path_factory):
    cfg, seed, page = H.CONFIGS[request.param]
    folder = str(tmp_path_factory.mktemp(f"c8_{request.param}"))
    H.make_model(folder, cfg, seed)
    return {"name": request.param, "cfg": cfg, "folder": folder, "page": page}


def session(model, dtype, kv, poison=True, pages=40, **kw):
    from servelab_b200.replay import TraceSession
    return TraceSession(model["folder"], dtype, pages * model["page"], page_size=model["page"], max_live=4, poison_cache=poison,
                        kv_cache_dtype=kv, **kw)


# ------------------------------------------------------------------------------------------------------------ the mixer
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("kv", ["int8", "e4m3"])
@pytest.mark.parametrize("dim,rotary,window,bias", [(32, 32, None, True), (64, 32, None, True), (128, 128, 7, False), (40, 0, 5, True)])
def test_mixer_over_an_8_bit_cache(dtype, kv, dim, rotary, window, bias):
    from servelab_b200.config import AttentionSpec, NoPositionSpec, RotarySpec
    from servelab_b200.engine.batch import BatchEntry, StepContext
    from servelab_b200.ops import kernels as K
    from servelab_b200.parts import MIXERS, BuildEnv, LayerCache, build_part, part_class
    from servelab_b200.weights import RandomSource, WeightStore
    heads, kvh, hid, T, ps = 6, 2, 40, 29, 4
    spec = AttentionSpec(hidden_size=hid, num_heads=heads, num_kv_heads=kvh, head_dim=dim, qkv_bias=bias, out_bias=False, window=window,
                         position=RotarySpec(head_dim=dim, rotary_dim=rotary, theta=1e4) if rotary else NoPositionSpec())
    decls = part_class(MIXERS, spec).declare(spec, "a")
    src = RandomSource(decls, 3, std=0.08, dtype=DT[dtype])
    part = build_part(MIXERS, spec, "a", BuildEnv(device=DEV, dtype=DT[dtype], page_size=ps))
    part.load(WeightStore(src, decls, DT[dtype], DEV))
    w = {d.name: src.read(d.name).double() for d in decls}
    torch.manual_seed(5)
    x = torch.randn(T, hid).to(DT[dtype])

    def projected(name, n):
        y = P.linear(x.double(), w[f"a.{name}_proj.weight"], w.get(f"a.{name}_proj.bias")).view(T, n, dim)
        if name != "v" and rotary:
            turned = P.rope(y[..., :rotary], torch.arange(T), P.rope_inv_freq(rotary, 1e4).double())
            y = torch.cat([turned, y[..., rotary:]], -1)
        return y.double()

    q, k, v = projected("q", heads), projected("k", kvh), projected("v", kvh)
    loose = {"float32": 1e-5, "bfloat16": 2e-2}[dtype]     # (the parts' own tests: roundings of the projections and the result)
    pages = [5, 0, 7, 3, 9, 1, 8, 2]
    for cuts in ([T], [3, 2, 11, 1, 1, 9, 2]):
        codes = torch.full((2, 10, kvh, ps, dim), 0x7E, dtype=torch.uint8, device=DEV).view(KINDS[kv])
        scales = torch.full((2, 10, kvh, ps), 1e25, device=DEV)
        cache = LayerCache(group=0, k=codes[0], v=codes[1], page_size=ps, k_scale=scales[0], v_scale=scales[1])
        outs, start = [], 0
        for n in cuts:
            ctx = StepContext.pack([BatchEntry([0] * n, start, (), [pages[:-(-(start + n) // ps)]])], 1, DEV)
            outs.append(K.plain_unless(None, part.forward(ctx, x[start:start + n].to(DEV), cache, True)).double().cpu())
            start += n
        got = torch.cat(outs)
        kc, vc = torch.empty(T, kvh, dim, device=DEV), torch.empty(T, kvh, dim, device=DEV)
        i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=DEV)
        K.cache_read(cache.k, cache.v, cache.k_scale, cache.v_scale, i32([pages]), i32([0]), i32([0, T]), ps, kc, vc)
        kc, vc = kc.double().cpu(), vc.double().cpu()
        for back, row in ((kc, k), (vc, v)):
            top = row.abs().amax(-1, keepdim=True)
            half = top / 254 if kv == "int8" else row.abs() / 16 + top / 448 / 1024
            assert bool(((back - row).abs() <= 1.01 * half + loose).all())
        want = P.linear(P.causal_attention(q, kc, vc, window).double(), w["a.o_proj.weight"])
        assert (got - want).abs().max() <= loose, (cuts, float((got - want).abs().max()))


# ----------------------------------------------------------------------------------------------------------- whole models
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("kv", ["int8", "e4m3"])
def test_steps_with_an_8_bit_cache(model, dtype, kv):
    """Logits near the plain implementation's, and the very same ones whatever unwritten slots hold."""
    requests = {f"r{i}": H.random_ids(n, model["cfg"]["vocab_size"], 50 + i) for i, n in enumerate([70, 45, 97, 33, 58])}
    steps = H.trace_mixed(requests, 3)
    vocab = model["cfg"]["vocab_size"]
    got = H.collect(steps, H.run_session(session(model, dtype, kv), steps), vocab)
    clean = H.collect(steps, H.run_session(session(model, dtype, kv, poison=False), steps), vocab)
    worst = 0.0
    for rid, ids in requests.items():
        want = H.plain_logits(model["folder"], ids)
        for j, row in got[rid].items():
            assert np.array_equal(row, clean[rid][j]), (rid, j)
            worst = max(worst, float(np.abs(row - want[j]).max()))
    print(model["name"], dtype, kv, worst)
    assert worst <= tol(model["name"], dtype, kv)


def random_tree(n, rng):
    return [-1 if j == 0 or rng.random() < 0.2 else rng.randint(max(0, j - 4), j - 1) for j in range(n)]


def path(parents, j):
    out = []
    while j >= 0:
        out.append(j)
        j = parents[j]
    return out[::-1]


@pytest.mark.parametrize("kv", ["auto", "int8"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_drafted_trees_get_the_logits_of_their_paths(model, dtype, kv):
    """Two trees and a plain token in one step, every token against its own path; then an accepted path sent again as the head of
    the next trees, against paths behind it.  (The cache is poisoned; rejected drafts lie in it when the second step runs.)"""
    rng = random.Random(7)
    vocab, limit = model["cfg"]["vocab_size"], tol(model["name"], dtype, kv)
    prompts = {"a": H.random_ids(37, vocab, 1), "b": H.random_ids(60, vocab, 2), "c": H.random_ids(20, vocab, 3)}
    sess = session(model, dtype, kv)
    sess.run_step({"entries": [{"id": r, "tokens": ids} for r, ids in prompts.items()]})
    held = {r: list(ids) for r, ids in prompts.items()}
    head = {"a": [], "b": []}
    worst = 0.0
    for sizes in ({"a": 13, "b": 40}, {"a": 6, "b": 9}):
        entries, asked = [], []
        for r, n in sizes.items():
            keep = len(head[r])
            tree = list(range(-1, keep - 1)) + [p + keep if p >= 0 else keep - 1 for p in random_tree(n, rng)]
            tokens = head[r] + H.random_ids(n, vocab, rng.randint(0, 999))
            entries.append({"id": r, "tokens": tokens, "parents": tree, "keep": keep, "want": list(range(len(tokens)))})
            asked += [held[r] + [tokens[i] for i in path(tree, j)] for j in range(len(tokens))]
            deepest = max(range(len(tokens)), key=lambda j: len(path(tree, j)))
            held[r] += head[r]
            head[r] = [tokens[i] for i in path(tree, deepest)][keep:]
        one = H.random_ids(1, vocab, rng.randint(0, 999))
        entries.insert(1, {"id": "c", "tokens": one, "want": [0]})
        held["c"] += one
        asked.insert(len(entries[0]["tokens"]), list(held["c"]))
        got = sess.run_step({"entries": entries})
        assert got.shape[0] == len(asked)
        for row, ids in zip(got, asked):
            worst = max(worst, float(np.abs(row - H.plain_logits(model["folder"], ids)[-1]).max()))
        assert sess.held == {r: len(ids) for r, ids in held.items()}
    print(model["name"], dtype, kv, worst)
    assert worst <= limit


@pytest.mark.parametrize("kv", ["auto", "int8", "e4m3"])
def test_cached_rows_are_what_the_cache_holds(model, kv):
    sess = session(model, "bfloat16", kv)
    ids = H.random_ids(41, model["cfg"]["vocab_size"], 9)
    sess.run_step({"entries": [{"id": "x", "tokens": ids}]})
    cache, table = sess.runner.storage.layer_caches[0], sess.cache.block_table("x", sess.runner.storage.layer_caches[0].group)
    k, v = sess.runner.cached_rows("x", 30, start=5)
    assert k.shape == (30, model["cfg"]["num_key_value_heads"], model["cfg"]["head_dim"]) and k.dtype == torch.bfloat16
    for got, rows, scale in ((k, cache.k, cache.k_scale), (v, cache.v, cache.v_scale)):
        for i in range(30):
            page, slot = table[(5 + i) // model["page"]], (5 + i) % model["page"]
            want = rows[page, :, slot].float()
            if scale is not None:
                want = want * scale[page, :, slot][:, None]
            assert torch.equal(got[i], want.to(torch.bfloat16)), i
    with pytest.raises(ValueError):
        sess.runner.cached_rows("x", -1)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("kv", ["int8", "e4m3"])
def test_generation_with_and_without_graphs(model, dtype, kv):
    from servelab_b200.config import CacheConfig, SchedulerConfig
    from servelab_b200.engine.llm_engine import LLMEngine
    from servelab_b200.sampling import SamplingParams
    prompts = [H.random_ids(n, model["cfg"]["vocab_size"] - 2, 70 + n) for n in (5, 33, 61)]

    def tokens(**kw):
        eng = LLMEngine(model["folder"], CacheConfig(block_size=model["page"], num_blocks=64, kv_cache_dtype=kv, poison_cache=True),
                        SchedulerConfig(max_num_seqs=8, max_num_batched_tokens=24), dtype=dtype, **kw)
        eng.runner.portion_graph_after = 1
        outs = eng.generate(prompts, SamplingParams(temperature=0.0, max_tokens=10, ignore_eos=True))
        return [o.outputs[0].token_ids for o in outs], eng

    got, eng = tokens()
    assert eng.runner.graph_replays > 0 and eng.runner.portion_graph_replays > 0
    assert eng.runner.storage.layer_caches[0].k.dtype == KINDS[kv]
    assert got == tokens(cuda_graphs=False)[0]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("kv", ["auto", "int8"])
def test_far_drafts_leave_the_keys_that_decoding_leaves(model, dtype, kv):
    """The first layer's keys and values at slots around 30,000 (they go by token and position alone), written by a step of
    single tokens, by a portion of a prompt and by a tree that is a chain: the very same rows."""
    start, n = 30001, 5
    ids = H.random_ids(n, model["cfg"]["vocab_size"], 77)
    sess = session(model, dtype, kv, poison=False, pages=-(-(start + 64) // model["page"]))
    runner = sess.runner
    written = {}
    for how in ("single", "portion", "tree"):
        assert runner.cache.open(how)
        assert runner.cache.ensure(how, start + n)
        if how == "single":
            for j in range(n):
                runner.step([runner.entry(how, ids[j:j + 1], start + j, [0])])
        else:
            runner.step([runner.entry(how, ids, start, [n - 1], list(range(-1, n - 1)) if how == "tree" else None)])
        written[how] = runner.cached_rows(how, n, start=start)
        runner.cache.release(how)
    for how in ("portion", "tree"):
        for a, b in zip(written[how], written["single"]):
            # (float32 products do not depend on the step; bfloat16 steps of few tokens rotate before they round, and the products
            # of different sizes add up in different orders: two roundings apart, or a code)
            if dtype == "float32":
                assert torch.equal(a, b), how
            else:
                top = b.float().abs().amax(-1, keepdim=True)
                assert ((a.float() - b.float()).abs() <= 2.0 ** -7 * b.float().abs() + (2.0 ** -6 if kv == "int8" else 2.0 ** -8) * top).all(), how


@pytest.mark.parametrize("kv", ["int8", "e4m3"])
@pytest.mark.parametrize("name", ["D", "E"])
def test_replayed_steps_planned_for_long_contexts(name, kv, tmp_path):
    """Decode steps replay a graph whose launches were chosen for 32,768 keys (head sizes 64 and 128): logits near those of steps
    that are planned for their own contexts, which are short."""
    cfg, seed, page = H.CONFIGS[name]
    long = {"name": name, "cfg": {**cfg, "max_position_embeddings": 32768}, "folder": str(tmp_path), "page": page}
    H.make_model(long["folder"], long["cfg"], seed, std_of=H.STD_OF.get(name))
    requests = {f"r{i}": H.random_ids(n, cfg["vocab_size"], 80 + i) for i, n in enumerate([70, 33, 58])}
    steps = H.trace_bulk_tail(requests, tail=12)
    got = {}
    for graphs in (True, False):
        sess = session(long, "bfloat16", kv, pages=32768 // page + 4, cuda_graphs=graphs)
        assert sess.runner.max_model_len == 32768
        got[graphs] = H.collect(steps, H.run_session(sess, steps), cfg["vocab_size"])
        assert (sess.runner.graph_replays > 0) == graphs
    # (two sums in other orders of the same codes: roundings of bfloat16, as the bounds of a cache in that type)
    far = max(float(np.abs(row - got[False][r][j]).max()) for r in requests for j, row in got[True][r].items())
    assert far <= TOL["bfloat16"][name]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("kv", ["int8", "e4m3"])
@pytest.mark.parametrize("far", [0, 4000])
def test_mixer_that_reads_anothers_8_bit_cache(dtype, kv, far):
    """A run without a cache of its own: its queries over the rows that another run left, also at far positions."""
    from servelab_b200.config import AttentionSpec, RotarySpec
    from servelab_b200.engine.batch import BatchEntry, StepContext
    from servelab_b200.ops import kernels as K
    from servelab_b200.parts import MIXERS, BuildEnv, LayerCache, build_part, part_class
    from servelab_b200.weights import RandomSource, WeightStore
    heads, kvh, hid, T, ps, dim = 6, 2, 40, 21, 16, 64
    spec = AttentionSpec(hidden_size=hid, num_heads=heads, num_kv_heads=kvh, head_dim=dim, qkv_bias=True, out_bias=False, window=T,
                         position=RotarySpec(head_dim=dim, rotary_dim=dim, theta=1e4))
    decls = part_class(MIXERS, spec).declare(spec, "a")
    parts, weights = [], []
    for seed in (3, 4):
        src = RandomSource(decls, seed, std=0.08, dtype=DT[dtype])
        parts.append(build_part(MIXERS, spec, "a", BuildEnv(device=DEV, dtype=DT[dtype], page_size=ps)))
        parts[-1].load(WeightStore(src, decls, DT[dtype], DEV))
        weights.append({d.name: src.read(d.name).double() for d in decls})
    torch.manual_seed(6)
    x = torch.randn(T, hid).to(DT[dtype])
    first = far // ps
    pages = [-1] * first + [3, 0, 2]
    codes = torch.zeros((2, 4, kvh, ps, dim), dtype=torch.uint8, device=DEV).view(KINDS[kv])
    scales = torch.zeros((2, 4, kvh, ps), device=DEV)
    cache = LayerCache(group=0, k=codes[0], v=codes[1], page_size=ps, k_scale=scales[0], v_scale=scales[1])
    ctx = StepContext.pack([BatchEntry([0] * T, first * ps, (), [pages])], 1, DEV)
    parts[0].forward(ctx, x.to(DEV), cache, True)
    before = [t.clone() for t in (codes.view(torch.uint8), scales)]
    got = K.plain_unless(None, parts[1].forward(ctx, x.to(DEV), cache, False)).double().cpu()
    assert torch.equal(codes.view(torch.uint8), before[0]) and torch.equal(scales, before[1])
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=DEV)
    kc, vc = torch.empty(T, kvh, dim, device=DEV), torch.empty(T, kvh, dim, device=DEV)
    K.cache_read(cache.k, cache.v, cache.k_scale, cache.v_scale, i32([pages]), i32([first * ps]), i32([0, T]), ps, kc, vc)
    w = weights[1]
    q = P.linear(x.double(), w["a.q_proj.weight"], w["a.q_proj.bias"]).view(T, heads, dim)
    # angles are float32 products of position and frequency, by definition
    angle = (torch.arange(first * ps, first * ps + T).float()[:, None] * P.rope_inv_freq(dim, 1e4).float()[None]).double()
    a, b = q[..., :dim // 2], q[..., dim // 2:]
    q = torch.cat([a * angle.cos()[:, None] - b * angle.sin()[:, None], b * angle.cos()[:, None] + a * angle.sin()[:, None]], -1)
    # (far on, slots of the window before the first token have no page: keys and values of zeros, which count)
    zeros = T if far else 0
    kc, vc = (torch.cat([torch.zeros(zeros, kvh, dim), t.cpu()]).double() for t in (kc, vc))
    q = torch.cat([torch.zeros(zeros, heads, dim).double(), q])
    want = P.linear(P.causal_attention(q, kc, vc, T).double()[zeros:], w["a.o_proj.weight"])
    assert (got - want).abs().max() <= {"float32": 1e-5, "bfloat16": 2e-2}[dtype]
