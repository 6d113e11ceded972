"""Each form of the attention over a cache by its name, at the inputs where its numbers can go wrong: value scales and
queries of far magnitudes in one tile, windows, peaked scores, infinities and NaN beside finite rows.  The form is forced, so that
small sizes reach the kernel for many rows; bounds are those of ``cache8_cases.bound``."""

import math

import pytest
import torch

import cache8_cases as C
import test_gpu_cache8 as B

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
# (form, blocks that share the keys, units with one more, blocks of a cluster, rows a block)
FORMS = {"tc": ("tc", 1, 0, 1, 0), "tc3": ("tc", 3, 0, 1, 0), "tc+": ("tc", 1, 3, 1, 0), "few8": ("few", 1, 0, 2, 8),
         "few16": ("few", 2, 0, 4, 16), "plain": ("plain", 2, 0, 1, 0)}


@pytest.fixture
def force(monkeypatch):
    """``force(name)``: attention runs in that form from here on; the returned list names the form of every call."""
    def forced(name):
        form, parts, more, cluster, block = FORMS[name]
        calls = []

        def plan(fast, kind, tokens, requests, group, num_kv_heads, head_dim, longest_q, longest):
            assert fast or form == "plain"
            calls.append(form)
            if form == "tc":
                tiles = tokens * group // 128 + requests
                return form, tiles, parts, min(more, tiles * num_kv_heads), 1, 0
            return form, -(-longest_q * group // (block or 8)), parts, 0, cluster, block

        monkeypatch.setattr(B.K(), "cache_attention_plan", plan)
        return calls
    return forced


def chain(s):
    """A mask under which every token sees what it sees causally."""
    words = max(1, -(-max(s["q_lens"]) // 32))
    bits = [(2 << j) - 1 for n in s["q_lens"] for j in range(n)]
    rows = [[b >> 32 * w & 0xFFFFFFFF for w in range(words)] for b in bits]
    positions = [c - n + j for n, c in zip(s["q_lens"], s["ctxs"]) for j in range(n)]
    rest = s["q"].shape[0] - len(bits)                     # (rows behind the last request's)
    rows, positions = rows + [[0] * words] * rest, positions + [0] * rest
    return C.i32([[w - (1 << 32) if w >> 31 else w for w in row] for row in rows], DEV), C.i32(positions, DEV), bits, positions


def attend_and_check(s, window=0):
    """Causal; a cache in the compute type by way of a mask that says the same."""
    if s["kind"] == "plain":
        mask, positions, bits, at = chain(s)
        B.attend(s, window=window, mask=mask, positions=positions)
        B.check(s, window=window, bits=bits, positions=at)
    else:
        B.attend(s, window=window)
        B.check(s, window=window)


def place(s, slot, request=0):
    page, at = divmod(slot, s["page"])
    return s["table"][request, page].item(), at


def set_row(s, name, slot, code, scale):
    """One cached row of all kv heads: every element the code of that number, and its scale."""
    page, at = place(s, slot)
    row = torch.full((s["kv"], s["dim"]), float(code), device=DEV).to(s[name].dtype)
    s[name].view(torch.uint8)[page, :, at] = row.view(torch.uint8)
    s[name + "s"][page, :, at] = scale


def leaning(kind, dim, q_lens, ctxs, seed):
    """A step whose queries have a common part along (1, .., 1), so that a key along it has about one score for all of them;
    and the scale with which a key of largest codes has the score 1 (natural units) there."""
    s = B.step("bfloat16", kind, 14, 2, dim, q_lens, ctxs, 16, seed=seed)
    s["q"].copy_((0.1 * s["q"].float() + 1.0).to(torch.bfloat16))
    return s, 1.0 / (dim * C.LARGEST[kind] * s["scale"])


FAST = ["tc", "tc3", "tc+", "few8", "few16"]


@pytest.mark.parametrize("form", FAST)
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("slot", [2, 130, 389, 393])
def test_a_large_value_row_of_no_weight(force, form, kind, dim, slot):
    """Its scale is 2^30 times the others', its weight 2^-60 of theirs: it adds 2^-30 and must cost the others nothing.  In the
    first tile, in one that all rows see, and among the step's own tokens (389: before the first row's, 393: seen by some)."""
    calls = force(form)
    s, one = leaning(kind, dim, [9], [400], 41)
    set_row(s, "k", slot, -C.LARGEST[kind], 60 * math.log(2) * one)
    page, at = place(s, slot)
    s["vs"][page, :, at] *= 2.0 ** 30
    attend_and_check(s)
    assert calls == [FORMS[form][0]]


@pytest.mark.parametrize("form", FAST)
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("slot", [2, 130, 389, 393])
def test_a_key_that_takes_all_weight_and_has_no_value(force, form, kind, dim, slot):
    """A first token that all others look at, its value row zeros: the result is what the others add, 2^-40 of theirs."""
    calls = force(form)
    s, one = leaning(kind, dim, [9], [400], 42)
    set_row(s, "k", slot, C.LARGEST[kind], 40 * math.log(2) * one)
    set_row(s, "v", slot, 0, C.TINY)
    attend_and_check(s)
    assert calls == [FORMS[form][0]]


@pytest.mark.parametrize("form", FAST + ["plain"])
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_value_scales_over_forty_powers_of_two(force, form, kind):
    calls = force(form)
    s = B.step("bfloat16", kind, 14, 2, 64, [19], [700], 16, seed=43)
    s["vs"] *= torch.exp2(torch.randint(-20, 21, s["vs"].shape, generator=B.gen(44), device=DEV).float())
    for factor in (1.0, 2.0 ** 80, 2.0 ** -90):
        attend_and_check({**s, "vs": s["vs"] * factor})
    for factor in (2.0 ** 60, 2.0 ** -60, 2.0 ** 120, 2.0 ** 125):
        attend_and_check({**s, "q": (s["q"].float() * factor).to(torch.bfloat16), "ks": s["ks"] / factor})
    assert set(calls) == {FORMS[form][0]}


@pytest.mark.parametrize("form", FAST)
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_value_scales_near_the_largest_that_count(force, form, kind):
    """All scales from 2^104 to 2^110: values of up to 2^117 (int8) or 2^118."""
    force(form)
    s = B.step("bfloat16", kind, 14, 2, 64, [5], [300], 16, seed=45)
    scale = torch.exp2(104 + 5.9 * torch.rand(s["vs"].shape, generator=B.gen(46), device=DEV))
    attend_and_check({**s, "vs": torch.where(torch.isnan(s["vs"]), s["vs"], scale)})


@pytest.mark.parametrize("form", FAST + ["plain"])
@pytest.mark.parametrize("kind", ["plain", "int8", "e4m3"])
@pytest.mark.parametrize("dim,window", [(64, 0), (128, 0), (128, 1), (64, 20), (128, 130)])
def test_portions_and_windows(force, form, kind, dim, window):
    calls = force(form)
    s = B.step("bfloat16", kind, 14, 2, dim, [5, 0, 33, 1, 70], [5, 0, 200, 77, 331], 16, seed=47, pad=1)
    attend_and_check(s, window)
    assert calls == [FORMS[form][0]]


@pytest.mark.parametrize("form", FAST)
@pytest.mark.parametrize("kind", ["plain", "int8", "e4m3"])
@pytest.mark.parametrize("page", [1, 5, 64])
def test_pages_of_any_size(force, form, kind, page):
    force(form)
    attend_and_check(B.step("bfloat16", kind, 14, 2, 64, [21, 3], [200, 131], page, seed=48), 40)


@pytest.mark.parametrize("form", FAST)
@pytest.mark.parametrize("kind", ["plain", "int8", "e4m3"])
@pytest.mark.parametrize("dim", [64, 128])
def test_peaked_scores(force, form, kind, dim):
    """Scores of some tens: references move in most tiles."""
    force(form)
    attend_and_check(B.step("bfloat16", kind, 14, 2, dim, [30, 1], [901, 300], 16, seed=49, spread=6.0))


def one_takes_all(s, q):
    """(tokens, heads) whose best key leads by more than scores may be off (twice (D + 3) 2^-24 of their products' magnitudes) and
    30 besides, and the value of that key [tokens, heads, D]."""
    n, c, heads, dim = s["q_lens"][0], s["ctxs"][0], s["heads"], s["dim"]
    k, v = (C.rows_of(s[x], s[x + "s"], s["table"][0], s["page"], c).repeat_interleave(heads // s["kv"], 0) for x in ("k", "v"))
    q = q.view(n, heads, dim).transpose(0, 1).to(torch.float64)
    scores = (q @ k.transpose(1, 2) * s["scale"]).masked_fill(~C.visible(n, c).to(DEV), -math.inf)
    off = 2 * (dim + 3) * 2.0 ** -24 * (q.abs() @ k.abs().transpose(1, 2) * s["scale"]).amax(-1)
    best = scores.topk(2, -1)
    value = torch.gather(v, 1, best.indices[..., :1].expand(-1, -1, dim))
    return (best.values[..., 0] - best.values[..., 1] > 2 * off + 30).T, value.transpose(0, 1)


@pytest.mark.parametrize("form", FAST + ["plain"])
@pytest.mark.parametrize("kind", ["plain", "int8", "e4m3"])
@pytest.mark.parametrize("dim,far", [(64, 18), (128, 22), (64, 24), (128, 25), (64, 26), (128, 27), (64, 28), (128, 30), (64, 34), (128, 60)])
def test_scores_of_any_size(force, form, kind, dim, far):
    """Scores of about 2^far, also where all of them are negative: numbers throughout, and one key's value where float32 tells
    which; for value scales of different sizes."""
    force(form)
    s = B.step("bfloat16", kind, 14, 2, dim, [12], [300], 16, seed=54)
    s["q"] = (2.0 ** far * s["q"].float()).to(torch.bfloat16)
    below = {**s, "q": (s["q"].float().abs()).to(torch.bfloat16), "k": -s["k"].abs() if kind != "e4m3" else
             (s["k"].view(torch.uint8) | 0x80).view(s["k"].dtype)}
    for t in (s, below):
        for factor in (1.0,) if kind == "plain" else (1.0, 2.0 ** -20, 2.0 ** 10):
            u = {**t, "vs": None if kind == "plain" else t["vs"] * factor}
            attend_and_check(u)
            sure, value = one_takes_all(u, u["q"])
            assert sure.float().mean() > 0.75
            off = (u["out"].view(12, 14, dim).to(torch.float64) - value).abs()[sure]
            assert (off <= 2.0 ** -7 * value[sure].abs() + 1e-30).all()


@pytest.mark.parametrize("form", FAST)
@pytest.mark.parametrize("kind", ["plain", "int8", "e4m3"])
@pytest.mark.parametrize("dim,far", [(64, 14), (128, 16), (64, 17), (128, 20), (64, 34), (128, 34), (64, 60), (128, 100)])
def test_query_rows_of_very_different_size(force, form, kind, dim, far):
    """Tokens and heads whose queries are 2^far times their neighbours', above or below."""
    force(form)
    s = B.step("bfloat16", kind, 14, 2, dim, [23], [300], 16, seed=50)
    for heads in (slice(3, 14, 3), slice(1, 14, 2)):
        q = s["q"].float().view(23, 14, dim).clone()
        q[::2, heads] *= 2.0 ** far
        attend_and_check({**s, "q": q.view(23, 14 * dim).to(torch.bfloat16)})
        attend_and_check({**s, "q": (q.view(23, 14 * dim) * 2.0 ** -far).to(torch.bfloat16)})


def near(s, clean, rows, window=0, bits=None, positions=None):
    """The results of those rows (boolean [tokens, heads]) of a step's only request within their bounds; ``clean``: the step whose
    inputs they go by."""
    n, c, heads, dim = s["q_lens"][0], s["ctxs"][0], s["heads"], s["dim"]
    k, v = (C.rows_of(clean[x], clean[x + "s"], s["table"][0], s["page"], c) for x in ("k", "v"))
    want, mag, dots = C.attention(clean["q"].view(n, heads, dim), k, v, C.visible(n, c, window, bits, positions), s["scale"],
                                  heads // s["kv"])
    far = (s["out"].view(n, heads, dim).to(torch.float64) - want).abs() - C.bound(want, mag, dots, c, dim, True, torch.bfloat16)
    return bool((far[rows] <= 0).all())


def but(tokens, *none):
    rows = torch.ones(tokens, 14, dtype=torch.bool, device=DEV)
    for t in none:
        rows[t] = False
    return rows


@pytest.mark.parametrize("form", FAST + ["plain"])
@pytest.mark.parametrize("kind", ["plain", "int8", "e4m3"])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_a_query_row_that_is_not_finite(force, form, kind, bad):
    """Its own result is no number; the rows beside it are as without it."""
    force(form)
    s = B.step("bfloat16", kind, 14, 2, 64, [12], [300], 16, seed=51)
    t = {**s, "q": s["q"].clone()}
    t["q"].view(12, 14, 64)[4, 5, 17] = bad
    if kind == "plain":
        mask, positions, _, _ = chain(s)
        B.attend(t, mask=mask, positions=positions)
    else:
        B.attend(t)
    assert torch.isnan(t["out"].view(12, 14, 64)[4, 5].float()).all()
    assert near(t, s, but(12, (4, 5)))


@pytest.mark.parametrize("form", FAST + ["plain"])
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_scales_of_rows_that_are_not_seen(force, form, kind):
    """NaN and infinite scales of a draft on another branch, of slots behind a causal token and before a window."""
    force(form)
    s = B.step("bfloat16", kind, 14, 2, 64, [6], [140], 16, seed=52)
    page, at = place(s, 134 + 3)                           # drafted token 3: seen by itself alone
    bits, where = [1, 3, 7, 15, 17, 49], list(range(134, 140))
    for k_scale, v_scale in ((math.nan, math.inf), (math.inf, math.nan), (math.nan, 1.0), (1.0, math.nan)):
        t = {**s, "ks": s["ks"].clone(), "vs": s["vs"].clone()}
        t["ks"][page, :, at], t["vs"][page, :, at] = k_scale, v_scale
        B.attend(t, mask=C.i32([[b] for b in bits], DEV), positions=C.i32(where, DEV))
        assert near(t, s, but(6, 3), bits=bits, positions=where)
        none = torch.isnan(t["out"][3].float()).all()
        B.attend(t)                                        # causal: tokens 3, 4 and 5 see it
        assert near(t, s, but(6, 3, 4, 5))
        # (infinite keys and NaN values: a score of -inf may leave the value out)
        assert math.isinf(k_scale) or none and torch.isnan(t["out"][3:].float()).all()
    page, at = place(s, 70)                                # before the window of every token
    t = {**s, "ks": s["ks"].clone(), "vs": s["vs"].clone()}
    t["ks"][page, :, at], t["vs"][page, :, at] = math.nan, math.nan
    B.attend(t, window=50)
    assert near(t, s, but(6), window=50)


@pytest.mark.parametrize("form", FAST + ["plain"])
@pytest.mark.parametrize("kind", ["plain", "int8", "e4m3"])
def test_the_same_bits_every_time(force, form, kind):
    force(form)
    s = B.step("bfloat16", kind, 14, 2, 128, [40, 1], [1500, 700], 16, seed=53)
    attend_and_check(s)
    first = s["out"].clone()
    mask, positions, _, _ = chain(s)
    for _ in range(20):
        s["out"].fill_(3.0)
        if kind == "plain":
            B.attend(s, mask=mask, positions=positions)
        else:
            B.attend(s)
        assert torch.equal(s["out"], first)


@pytest.mark.parametrize("kind", ["plain", "int8", "e4m3"])
@pytest.mark.parametrize("dim,tokens", [(64, 1), (128, 40)])
@pytest.mark.parametrize("which", ["k", "v"])
def test_caches_that_begin_anywhere(kind, dim, tokens, which):
    """A cache that is a view from an odd element on: the plain kernel takes it, as it is promised."""
    s = B.step("bfloat16", kind, 14, 2, dim, [tokens, 2], [300, 90], 16, seed=55)
    flat = torch.empty(s[which].numel() + 1, dtype=s[which].dtype, device=DEV)
    view = flat[1:].view(s[which].shape)
    view.copy_(s[which])
    assert view.data_ptr() % 16 != 0 and view.is_contiguous()
    attend_and_check({**s, which: view})
    s["out"].fill_(7.0)
    attend_and_check(s)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("heads,kv,dim,rotary", [(14, 2, 64, 64), (4, 2, 128, 64), (5, 5, 20, 12), (4, 2, 48, 48)])
def test_rows_with_the_angles_of_other_writers(dtype, heads, kv, dim, rotary):
    """``cache_write`` without exact angles leaves what ``qkv_rope_cache`` leaves, at any position; and with codes what rows that
    it has turned (exactly, in float32) become as codes."""
    w = B.write_case(dtype, "plain", heads, kv, dim, rotary, [7, 33], [130001, 30000], 16, seed=dim)
    other = {n: torch.zeros_like(w[n]) for n in ("q_out", "k", "v")}
    args = (w["qkv"], w["bias"], w["positions"])
    B.K().qkv_rope_cache(*args, w["seq"], w["table"], 16, w["inv"], rotary, other["q_out"], other["k"], other["v"], heads, kv, dim)
    B.K().cache_write(*args, None, w["seq"], w["table"], 16, w["inv"], rotary, w["q_out"], w["k"], w["v"], None, None, heads, kv, dim,
                      exact_angles=False)
    for n in other:
        assert torch.equal(w[n], other[n]), n
    if dtype == "float32":
        codes = [torch.zeros(w["k"].shape, dtype=torch.int8, device=DEV) for _ in range(2)]
        scales = [torch.zeros(w["k"].shape[:3], device=DEV) for _ in range(2)]
        B.K().cache_write(*args, None, w["seq"], w["table"], 16, w["inv"], rotary, w["q_out"], *codes, *scales, heads, kv, dim,
                          exact_angles=False)
        for rows, code, scale in zip((w["k"], w["v"]), codes, scales):
            want = rows.abs().amax(-1) / 127               # (a product with 1 / 127 or a division: a unit apart at most)
            assert ((scale - want).abs() <= 2.0 ** -22 * want)[want > 0].all()
            # half a code, and what the scale's reciprocal and the product round
            assert ((code * scale[..., None] - rows).abs() <= (0.5 + 2.0 ** -14) * scale[..., None]).all()


@pytest.mark.parametrize("form", FAST + ["plain"])
@pytest.mark.parametrize("kind", ["plain", "int8"])
@pytest.mark.parametrize("window", [0, 90])
def test_a_tree_beside_a_long_portion(force, form, kind, window):
    """A portion of 331 tokens as a chain and a tree of 37 drafts in one step: eleven words of a mask."""
    from servelab_b200.engine.batch import tree_depths, tree_mask
    force(form)
    q_lens, ctxs = [331, 37, 1], [400, 200, 90]
    trees = [range(-1, 330), B.parents_of(37, 5), [-1]]
    s = B.step("bfloat16", kind, 4, 2, 64, q_lens, ctxs, 16, seed=56, pad=2)
    words = tree_mask(trees)
    bits = [sum((int(w) & 0xFFFFFFFF) << 32 * i for i, w in enumerate(row)) for row in words]
    positions = [c - n + d for n, c, t in zip(q_lens, ctxs, trees) for d in tree_depths(t)]
    mask = torch.cat([torch.from_numpy(words).to(DEV), torch.full((2, words.shape[1]), -1, dtype=torch.int32, device=DEV)])
    B.attend(s, window=window, mask=mask, positions=C.i32(positions + [0, 0], DEV))
    B.check(s, window=window, bits=bits, positions=positions)
